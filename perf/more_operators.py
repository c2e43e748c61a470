"""Measured cases of the experts' products, the row norm and the optimizer step, with their plain forms.

What a routed layer computes between dispatch and combine, and what trains it: the
gated feed-forward of rows sorted by expert and the plain product that follows it
(each with its gradients), the root-mean-square norm of rows with the residual's
addition (its output of the rows' type or in 8 bits with scales, and its gradients),
and one AdamW step over many tensors with states in 32 or in 8 bits.  ``run`` makes
one pass: in elementary torch operations in 32 bits, or with the framework's own
calls when ``own`` is true.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
E4M3_MOST = 448.0
GROUP = 32  # columns of a row that share a scale
BLOCK = 256  # elements of an optimizer state that share a scale
EPS = 1e-6
BETAS, ADAM_EPS, RATE, DECAY, STEPS = (0.9, 0.999), 1e-8, 1e-3, 0.1, 100  # an ordinary training step


def listed():
    return [
        # one token of a decode step, two experts: latency
        {"name": "gated_token", "kind": "gated", "rows": 2, "experts": 16, "width": 2048, "hidden": 1024,
         "dtype": "bf16", "activation": "silu", "balanced": False, "behind": 0.0},
        # a ragged serving batch whose router leaves some entries without an expert
        {"name": "gated_ragged", "kind": "gated", "rows": 3111, "experts": 37, "width": 1000, "hidden": 616,
         "dtype": "f16", "activation": "gelu", "balanced": False, "behind": 0.05},
        # the prompts of a serving batch, four experts a token
        {"name": "gated_prompt", "kind": "gated", "rows": 131072, "experts": 64, "width": 2048, "hidden": 1024,
         "dtype": "bf16", "activation": "silu", "balanced": False, "behind": 0.0},
        # gradients of a small layer in 32 bits, odd sizes
        {"name": "gated_grad_odd", "kind": "gated_grad", "rows": 8198, "experts": 8, "width": 257, "hidden": 129,
         "dtype": "f32", "activation": "silu", "balanced": False, "behind": 0.02},
        # gradients of one layer in a training step, rows split evenly by exact balanced transport
        {"name": "gated_grad_train", "kind": "gated_grad", "rows": 65536, "experts": 32, "width": 2048, "hidden": 1024,
         "dtype": "bf16", "activation": "silu", "balanced": True, "behind": 0.0},
        # the way back to the rows' width for a decode batch of 64 tokens: bound by the weights
        {"name": "product_batch", "kind": "product", "rows": 512, "experts": 64, "width": 1024, "hidden": 2048,
         "dtype": "bf16", "balanced": False, "behind": 0.0},
        # its gradients in a training step
        {"name": "product_grad_train", "kind": "product_grad", "rows": 65536, "experts": 32, "width": 1024,
         "hidden": 2048, "dtype": "bf16", "balanced": True, "behind": 0.0},
        # the tokens of a decode step of a few requests, read on by products in 8 bits: latency
        {"name": "norm_token", "kind": "norm", "rows": 5, "width": 2048, "dtype": "bf16", "residual": True,
         "held": "8 bits"},
        # the tokens of long prompts
        {"name": "norm_prompt", "kind": "norm", "rows": 32768, "width": 2048, "dtype": "bf16", "residual": True,
         "held": "same"},
        # gradients in a training step, with the residual path's own
        {"name": "norm_grad_train", "kind": "norm_grad", "rows": 65536, "width": 2048, "dtype": "bf16",
         "residual": True},
        # a small model: matrices with odd sides and vectors
        {"name": "adamw_small", "kind": "adamw", "tensors": 14, "elements": 200_003, "dtype": "f32", "master": False,
         "bits": 32},
        # a large model: parameters in 16 bits with 32-bit masters, states in 8 bits
        {"name": "adamw_train", "kind": "adamw", "tensors": 14, "elements": 400_000_000, "dtype": "bf16",
         "master": True, "bits": 8},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    width = _log(rng, low, high)
    return max(low, width // 8 * 8) if rng.random() < 0.5 else width


def draw(rng):
    kind = rng.choice(["gated", "gated", "gated_grad", "product", "product_grad", "norm", "norm_grad", "adamw", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("gated", "gated_grad", "product", "product_grad"):
        width, hidden = _width(rng, 16, 2048), _width(rng, 16, 2048)
        most = (1 << 37) // (4 if dtype == "f32" else 1)
        rows = min(_log(rng, 1 if kind in ("gated", "product") else 16, 131072), most // (width * hidden))
        case = {"kind": kind, "rows": rows, "experts": _log(rng, 1, 128), "width": width, "hidden": hidden,
                "dtype": dtype, "balanced": rng.random() < 0.5, "behind": rng.choice([0.0, 0.0, 0.1 * rng.random()])}
        if kind in ("gated", "gated_grad"):
            case["activation"] = rng.choice(["silu", "gelu"])
        return case
    if kind in ("norm", "norm_grad"):
        width = _width(rng, 16, 8192)
        rows = min(_log(rng, 1 if kind == "norm" else 16, 65536), (1 << 27) // width)
        case = {"kind": kind, "rows": rows, "width": width, "dtype": dtype, "residual": rng.random() < 0.7}
        if kind == "norm":
            case["held"] = rng.choice(["same", "8 bits"])
        return case
    return {"kind": kind, "tensors": rng.randint(1, 14), "elements": _log(rng, 1000, 200_000_000), "dtype": dtype,
            "master": dtype != "f32" and rng.random() < 0.7, "bits": rng.choice([8, 32])}


def _sizes(case):
    """Element counts of an optimizer step's tensors: a few large ones, many small ones, odd counts among them."""
    n, total = case["tensors"], case["elements"]
    shares = [1.0 / (1 + i % 5) ** 2 for i in range(n)]
    return [max(1, int(total * s / sum(shares)) - i % 3) for i, s in enumerate(shares)]


def _offsets(case, gen):
    """First row of each expert, int32: equal counts, or the uneven ones of a router; rows behind the last have none."""
    n, e = case["rows"], case["experts"]
    live = n - int(n * case["behind"])
    if case["balanced"]:
        return (torch.arange(e + 1, device="cuda") * live // e).to(torch.int32)
    lean = torch.randn(e, generator=gen, device="cuda") * 0.5
    chosen = torch.multinomial(torch.softmax(lean, 0), live, replacement=True, generator=gen)
    return torch.searchsorted(torch.sort(chosen).values, torch.arange(e + 1, device="cuda")).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]

    def normal(*shape, dtype=dtype):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    state = {"kind": kind}
    if kind in ("gated", "gated_grad", "product", "product_grad"):
        n, e, d, f = case["rows"], case["experts"], case["width"], case["hidden"]
        state["offsets"], state["x"] = _offsets(case, gen), normal(n, d)
        names = ("gate", "up") if kind in ("gated", "gated_grad") else ("weight",)
        state.update({name: normal(e, f, d).mul_(d ** -0.5) for name in names})
        if kind in ("gated", "gated_grad"):
            state["activation"] = case["activation"]
        if kind in ("gated_grad", "product_grad"):
            state["dy"] = normal(n, f)
    elif kind in ("norm", "norm_grad"):
        n, d = case["rows"], case["width"]
        state["x"], state["weight"] = normal(n, d), normal(d).mul_(0.1).add_(1.0)
        if kind == "norm":
            state["residual"], state["held"] = normal(n, d).mul_(2.0) if case["residual"] else None, case["held"]
        else:
            state["dy"], state["dsum"] = normal(n, d), normal(n, d) if case["residual"] else None
    else:
        sizes, bits = _sizes(case), case["bits"]
        full = [normal(n, dtype=torch.float32).mul_(0.02) for n in sizes]
        state["params"] = [p.to(dtype) for p in full]
        state["master"] = full if case["master"] else None
        state["grads"] = [normal(n).mul_(0.02) for n in sizes]
        state["norm"] = torch.tensor(0.02 * math.sqrt(sum(sizes)), device="cuda")
        state["limit"] = 0.5 * 0.02 * math.sqrt(sum(sizes))
        first = [normal(n, dtype=torch.float32).mul_(0.004) for n in sizes]
        second = [normal(n, dtype=torch.float32).mul_(0.01).square_() for n in sizes]
        state["first_scale"] = state["second_scale"] = None
        if bits == 8:
            first, state["first_scale"] = map(list, zip(*[_to_8_bits(v) for v in first]))
            second, state["second_scale"] = map(list, zip(*[_to_8_bits(v.sqrt_()) for v in second]))
        state["first"], state["second"] = first, second
        state["step"] = torch.tensor(STEPS, dtype=torch.int32, device="cuda")
    return state


def _run_own(s):
    import __graft_entry__ as entry
    hb = entry.load_package()
    kind = s["kind"]
    if kind == "gated":
        return {"h": hb.expert_gated(s["x"], s["gate"], s["up"], s["offsets"], activation=s["activation"])}
    if kind == "gated_grad":
        dx, dgate, dup = hb.expert_gated_grad(s["dy"], s["x"], s["gate"], s["up"], s["offsets"],
                                              activation=s["activation"])
        return {"dx": dx, "dgate": dgate, "dup": dup}
    if kind == "product":
        return {"y": hb.expert_product(s["x"], s["weight"], s["offsets"])}
    if kind == "product_grad":
        dx, dw = hb.expert_product_grad(s["dy"], s["x"], s["weight"], s["offsets"])
        return {"dx": dx, "dweight": dw}
    if kind == "norm":
        if s["held"] == "8 bits":
            rows, total = hb.rms_norm_8bit(s["x"], s["weight"], s["residual"], eps=EPS)
            out = {"y": hb.rows_of_8bit(rows, dtype=torch.bfloat16)}  # 4 bits and a power of two: exact
        elif s["residual"] is None:
            out, total = {"y": hb.rms_norm(s["x"], s["weight"], eps=EPS)}, None
        else:
            y, total = hb.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
            out = {"y": y}
        return {**out, "sum": total} if s["residual"] is not None else out
    if kind == "norm_grad":
        dx, dw = hb.rms_norm_grad(s["dy"], s["x"], s["weight"], dsum=s["dsum"], eps=EPS)
        return {"dx": dx, "dweight": dw}
    state = hb.AdamWState(s["first"], s["second"], s["first_scale"], s["second_scale"], s["master"], s["step"])
    hb.adamw_step(s["params"], s["grads"], state, lr=RATE, betas=BETAS, eps=ADAM_EPS, weight_decay=DECAY,
                  norm=s["norm"], max_norm=s["limit"])
    out = {"params": s["params"], "master": s["master"], "first": s["first"], "second": s["second"], "step": s["step"]}
    if s["first_scale"] is not None:
        out["first"], out["second"] = hb.adamw_moments(state)
    return out


def _activation(g, name):
    """(act(g), its derivative)."""
    if name == "silu":
        sig = 1.0 / (1.0 + torch.exp(-g))
        return g * sig, sig * (1.0 + g * (1.0 - sig))
    cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _by_expert(offsets, n):
    """The rows of each expert, padded to the longest: (rows [experts, longest], which of them there are, and the
    expert and place of each row)."""
    offsets = offsets.long()
    counts = offsets[1:] - offsets[:-1]
    place = torch.arange(max(1, int(counts.max())), device=offsets.device)
    rows = (offsets[:-1, None] + place).clamp(max=n - 1)
    row = torch.arange(n, device=offsets.device)
    expert = (torch.searchsorted(offsets, row, right=True) - 1).clamp(max=counts.numel() - 1)
    there = row < offsets[-1]
    return rows, place < counts[:, None], expert, torch.where(there, row - offsets[expert], 0), there


def _run_experts(s):
    kind, dtype = s["kind"], s["x"].dtype
    rows, live, expert, place, there = _by_expert(s["offsets"], s["x"].shape[0])
    zero = torch.zeros((), device=rows.device)

    def padded(v):
        return torch.where(live.unsqueeze(-1), v.float()[rows], zero)

    def back(v):
        return torch.where(there.unsqueeze(-1), v[expert, place], zero).to(dtype)

    x = padded(s["x"])
    if kind == "product":
        return {"y": back(torch.bmm(x, s["weight"].float().transpose(1, 2)))}
    if kind == "product_grad":
        dy = padded(s["dy"])
        return {"dx": back(torch.bmm(dy, s["weight"].float())), "dweight": torch.bmm(dy.transpose(1, 2), x).to(dtype)}
    gate, up = s["gate"].float(), s["up"].float()
    g, u = torch.bmm(x, gate.transpose(1, 2)), torch.bmm(x, up.transpose(1, 2))
    act, slope = _activation(g, s["activation"])
    if kind == "gated":
        return {"h": back(act * u)}
    dh = padded(s["dy"])
    dg, du = dh * u * slope, dh * act
    return {"dx": back(torch.bmm(dg, gate) + torch.bmm(du, up)), "dgate": torch.bmm(dg.transpose(1, 2), x).to(dtype),
            "dup": torch.bmm(du.transpose(1, 2), x).to(dtype)}


def _groups(y):
    """y [n, d] as [n, groups, GROUP], zeros behind its columns."""
    n, d = y.shape
    whole = -(-d // GROUP) * GROUP
    return torch.nn.functional.pad(y, (0, whole - d)).view(n, whole // GROUP, GROUP)


def _held_in_8_bits(y):
    """The values that y's 8-bit form stands for: groups of 32 columns share the smallest power of two by which their
    largest fits e4m3."""
    groups = _groups(y)
    most = groups.abs().amax(-1, keepdim=True)
    fraction, exponent = torch.frexp(most)  # fraction in [1/2, 1); 448 = 0.875 * 2^9
    exponent = (exponent - 9 + (fraction > 0.875)).clamp(-126, 127).to(torch.int32)
    unit = ((exponent + 127) << 23).view(torch.float32)
    held = (groups / unit).to(E4M3).float() * unit
    return held.view(y.shape[0], -1)[:, :y.shape[1]].to(torch.bfloat16)


def _to_8_bits(v):
    """(codes, scales): blocks of 256 elements share the scale that brings their largest to e4m3's."""
    n = v.numel()
    whole = -(-n // BLOCK) * BLOCK
    blocks = torch.nn.functional.pad(v, (0, whole - n)).view(-1, BLOCK)
    scale = blocks.abs().amax(1) / torch.full((), E4M3_MOST, device=v.device)
    return (blocks / torch.where(scale > 0, scale, 1.0)[:, None]).to(E4M3).view(-1)[:n], scale


def _of_8_bits(codes, scale):
    n = codes.numel()
    return codes.float() * scale.repeat_interleave(BLOCK)[:n]


def _root_to_8_bits(v):
    """The root of a second moment in 8 bits; one that is not zero keeps at least the smallest code."""
    codes, scale = _to_8_bits(v.sqrt())
    least = torch.full((), 2.0 ** -9, device=v.device).to(E4M3)
    return torch.where((v > 0) & (codes.float() == 0), least.float(), codes.float()).to(E4M3), scale


def _adamw(s, i, factor, rate, root):
    """One tensor's step, every operation rounded to 32 bits; returns what is held afterwards."""
    eight = s["first_scale"] is not None
    first, second = s["first"][i], s["second"][i]
    m = _of_8_bits(first, s["first_scale"][i]) if eight else first
    v = _of_8_bits(second, s["second_scale"][i]).square() if eight else second
    p = (s["params"] if s["master"] is None else s["master"])[i].float()
    g = s["grads"][i].float() * factor
    m = m * BETAS[0] + g * (1.0 - BETAS[0])
    v = v * BETAS[1] + (g * g) * (1.0 - BETAS[1])
    p = p * (1.0 - RATE * DECAY) - (m / (v.sqrt() / root + ADAM_EPS)) * rate
    if s["master"] is not None:
        s["master"][i].copy_(p)
    s["params"][i].copy_(p)
    if not eight:
        return first.copy_(m), second.copy_(v)
    codes, scale = _to_8_bits(m)
    first.copy_(codes), s["first_scale"][i].copy_(scale)
    codes, scale = _root_to_8_bits(v)
    second.copy_(codes), s["second_scale"][i].copy_(scale)
    return _of_8_bits(first, s["first_scale"][i]), _of_8_bits(second, s["second_scale"][i]).square()


def run(state):
    if own:
        return _run_own(state)
    s, kind = state, state["kind"]
    if kind in ("gated", "gated_grad", "product", "product_grad"):
        return _run_experts(s)
    if kind == "norm":
        total = s["x"].float() if s["residual"] is None else s["x"].float() + s["residual"].float()
        y = total * torch.rsqrt(total.square().mean(1, keepdim=True) + EPS) * s["weight"].float()
        out = {"y": _held_in_8_bits(y) if s["held"] == "8 bits" else y.to(s["x"].dtype)}
        return {**out, "sum": total.to(s["x"].dtype)} if s["residual"] is not None else out
    if kind == "norm_grad":
        x, dy = s["x"].float(), s["dy"].float()
        r = torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)
        wdy = dy * s["weight"].float()
        dx = r * wdy - x * (r * r * r * (wdy * x).mean(1, keepdim=True))
        if s["dsum"] is not None:
            dx = dx + s["dsum"].float()
        return {"dx": dx.to(s["x"].dtype), "dweight": (dy * x * r).sum(0).to(s["weight"].dtype)}
    s["step"].add_(1)
    t = s["step"].double()
    factor = (s["limit"] / (s["norm"].double() + 1e-6)).clamp(max=1.0).float()
    rate = (RATE / (1.0 - torch.pow(BETAS[0], t))).float()
    root = (1.0 - torch.pow(BETAS[1], t)).sqrt().float()
    moments = [_adamw(s, i, factor, rate, root) for i in range(len(s["params"]))]
    return {"params": s["params"], "master": s["master"], "first": [m for m, _ in moments],
            "second": [v for _, v in moments], "step": s["step"]}


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("gated", "gated_grad", "product", "product_grad"):
        ends = s["offsets"].tolist()
        n, d, f = case["rows"], case["width"], case["hidden"]
        zeros = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")  # noqa: E731
        forward = kind in ("gated", "product")
        out = zeros(n, f) if forward else zeros(n, d)
        grads = [] if forward else [zeros(case["experts"], f, d) for _ in range(2 if kind == "gated_grad" else 1)]
        for e, (a, b) in enumerate(zip(ends, ends[1:])):
            if a == b:
                continue
            x = s["x"][a:b].double()
            if kind == "product":
                out[a:b] = x @ s["weight"][e].double().t()
                continue
            if kind == "product_grad":
                dy = s["dy"][a:b].double()
                out[a:b] = dy @ s["weight"][e].double()
                grads[0][e] = dy.t() @ x
                continue
            gate, up = s["gate"][e].double(), s["up"][e].double()
            g, u = x @ gate.t(), x @ up.t()
            if case["activation"] == "silu":
                act = g * torch.sigmoid(g)
                slope = torch.sigmoid(g) * (1 + g * torch.sigmoid(-g))
            else:
                phi = torch.special.ndtr(g)
                act, slope = g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
            if kind == "gated":
                out[a:b] = act * u
                continue
            dh = s["dy"][a:b].double()
            dg, du = dh * u * slope, dh * act
            out[a:b] = dg @ gate + du @ up
            grads[0][e], grads[1][e] = dg.t() @ x, du.t() @ x
        names = {"gated": ["h"], "product": ["y"], "gated_grad": ["dx", "dgate", "dup"], "product_grad": ["dx", "dweight"]}
        return dict(zip(names[kind], [out, *grads]))
    if kind == "norm":
        total = s["x"].double() + (0.0 if s["residual"] is None else s["residual"].double())
        length = torch.linalg.vector_norm(total, dim=1, keepdim=True)
        y = total / (length * length / case["width"] + EPS).sqrt() * s["weight"].double()
        if case["held"] == "8 bits":  # the nearest of e4m3's values next to y, in the group's unit
            groups = _groups(y)
            unit = 2.0 ** torch.ceil(torch.log2(groups.abs().amax(-1, keepdim=True) / E4M3_MOST)).clamp(min=-126.0)
            ratio = groups / unit
            step = 2.0 ** (torch.floor(torch.log2(ratio.abs().clamp(min=2.0 ** -6))) - 3)
            y = (torch.round(ratio / step) * step * unit).view(case["rows"], -1)[:, :case["width"]]
        return {"y": y, "sum": total} if s["residual"] is not None else {"y": y}
    if kind == "norm_grad":
        x, dy, w = s["x"].double(), s["dy"].double(), s["weight"].double()
        rms = (torch.einsum("nd,nd->n", x, x) / case["width"] + EPS).sqrt()
        unit = x / rms[:, None]
        along = torch.einsum("nd,nd,d->n", dy, unit, w) / case["width"]
        dx = (dy * w - unit * along[:, None]) / rms[:, None]
        if s["dsum"] is not None:
            dx = dx + s["dsum"].double()
        return {"dx": dx, "dweight": torch.einsum("nd,nd->d", dy, unit)}
    t = STEPS + 1
    factor = min(1.0, s["limit"] / (float(s["norm"]) + 1e-6))
    params, firsts, seconds = [], [], []
    for i, p in enumerate(s["master"] or s["params"]):
        m, v = s["first"][i].double(), s["second"][i].double()
        if case["bits"] == 8:
            of = torch.arange(m.numel(), device="cuda") // BLOCK
            m, v = m * s["first_scale"][i].double()[of], (v * s["second_scale"][i].double()[of]) ** 2
        g = s["grads"][i].double() * factor
        m, v = BETAS[0] * m + (1 - BETAS[0]) * g, BETAS[1] * v + (1 - BETAS[1]) * g ** 2
        unbiased = m / (1 - BETAS[0] ** t), v / (1 - BETAS[1] ** t)
        params.append(p.double() - RATE * DECAY * p.double() - RATE * unbiased[0] / (unbiased[1].sqrt() + ADAM_EPS))
        firsts.append(m if case["bits"] == 32 else None)
        seconds.append(v if case["bits"] == 32 else None)
    return {"params": params, "master": params if s["master"] else None, "first": firsts, "second": seconds, "step": None}


def work(case):
    kind, size = case["kind"], DTYPES[case["dtype"]].itemsize
    if kind in ("gated", "gated_grad", "product", "product_grad"):
        n, e, d, f = case["rows"], case["experts"], case["width"], case["hidden"]
        live = n - int(n * case["behind"])
        # experts that have rows, where counts are even or nearly so
        named = min(e, live) if case["balanced"] else e * (1.0 - math.exp(live * math.log1p(-1.0 / e))) if e > 1 else 1
        mats = 2 if kind in ("gated", "gated_grad") else 1
        if kind in ("gated", "product"):
            return {"bytes": (live * d + n * f + mats * named * f * d) * size + 4 * (e + 1), "flops": 2 * mats * live * d * f}
        # gated: the products again, then to the rows and to the weights
        return {"bytes": (live * (d + f) + n * d + mats * (named + e) * f * d) * size + 4 * (e + 1),
                "flops": (6 if kind == "gated_grad" else 2) * 2 * live * d * f}
    if kind in ("norm", "norm_grad"):
        n, d = case["rows"], case["width"]
        if kind == "norm":
            out = 1 + 1 / GROUP + 2 if case["held"] == "8 bits" else size  # held, and its values read back
            return {"bytes": n * d * (size * (3 if case["residual"] else 1) + out) + d * size, "flops": 5 * n * d}
        return {"bytes": n * d * size * (4 if case["residual"] else 3) + 2 * d * size, "flops": 10 * n * d}
    n = sum(_sizes(case))
    held = 16 if case["bits"] == 32 else 2 * (2 + 8 / BLOCK) + 8  # read and written; in 8 bits their values too
    return {"bytes": n * (held + 2 * size + size * (0 if case["master"] else 1) + (8 if case["master"] else 0)), "flops": 15 * n}
