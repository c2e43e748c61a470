"""The experts', norm and optimizer calls together (examples/routed_block.py), and what they keep to beside their results on
ordinary arguments."""
import importlib.util
import sys
import threading
from pathlib import Path

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fw

import rows_reference as ref
from expert_reference import E23, activation

pytestmark = pytest.mark.gpu
EXAMPLES = Path(__file__).resolve().parents[1] / "examples"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("routed_block", EXAMPLES / "routed_block.py")
    module = importlib.util.module_from_spec(spec)
    sys.path.insert(0, str(EXAMPLES))
    try:
        spec.loader.exec_module(module)
    finally:
        sys.path.remove(str(EXAMPLES))
    return module


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.float16, 32), (torch.float32, 8), (torch.float32, 32)])
def test_training_steps_run(example, cuda, dtype, bits):
    for loss, norm in example.train(steps=3, tokens=200, experts=5, width=40, hidden=56, rows=60, dtype=dtype, bits=bits):
        assert np.isfinite(loss) and np.isfinite(norm) and norm > 0


def test_block_gradients_match_64_bits(example, hb, cuda):
    """Gradients of the whole fp32 block against the same block in 64-bit torch operations.  Every value passes fewer than
    16 sums of at most 128 terms, and the second norm divides by its rows' size, which is above 1/4 here:
    16 * 128 * 4 2^-24 of the largest gradient."""
    tokens, experts, width, hidden, rows = 150, 4, 48, 72, 40
    p = example.parameters(rows, experts, width, hidden, torch.float32)
    gen = torch.Generator(device=cuda).manual_seed(5)
    ids = torch.randint(0, rows, (tokens,), generator=gen, device=cuda)
    index = torch.randint(-1, experts, (tokens, 2), generator=gen, device=cuda)
    weights = torch.rand((tokens, 2), generator=gen, device=cuda)
    target = torch.randn((tokens, width), generator=gen, device=cuda)
    plan = hb.route_plan(index, experts)
    (example.block(hb, p, ids, plan, weights) - target).square().mean().backward()

    q = {k: v.detach().double().requires_grad_() for k, v in p.items()}

    def norm(t, w):
        return t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w

    x = q["table"][ids]
    n = norm(x, q["gain_in"])
    delta = torch.zeros_like(x)
    for k in range(2):
        live = (index[:, k] >= 0).nonzero().view(-1)
        e = index[live, k]
        g, u = (torch.einsum("td,thd->th", n[live], q[name][e]) for name in ("gate", "up"))
        z = torch.einsum("th,tdh->td", activation(g, "silu")[0] * u, q["down"][e])
        delta = delta.index_add(0, live, weights[live, k].double().unsqueeze(1) * z)
    t = x + delta
    assert float(t.square().mean(-1).min()) > 1 / 16
    (norm(t, q["gain_out"]) - target.double()).square().mean().backward()
    for name in p:
        got, want = p[name].grad, q[name].grad
        assert float((got.double() - want).abs().max()) <= 16 * 128 * 4 * 2.0 ** -24 * float(want.abs().max()), name


def _layer(hb, cuda, rows=300, dtype=torch.bfloat16, seed=1):
    gen = torch.Generator(device=cuda).manual_seed(seed)

    def normal(*size):
        return (torch.randn(size, generator=gen, device=cuda) * size[-1] ** -0.5).to(dtype)

    x, gain = normal(rows, 64), 1 + normal(64)
    first = torch.tensor([0, rows // 3, rows // 2, rows], dtype=torch.int32, device=cuda)
    return x, gain, normal(3, 128, 64), normal(3, 128, 64), normal(3, 64, 128), first


def _run(hb, x, gain, gate, up, down, first):
    y = hb.rms_norm(x, gain)
    return hb.rms_norm(hb.expert_product(hb.expert_gated(y, gate, up, first), down, first), gain, x)


def test_captured_forward_and_backward(hb, cuda):
    """A whole step captured into a graph and replayed on new values, next to an eager graph of other leaves."""
    args = _layer(hb, cuda)
    eager = [a.clone().requires_grad_() for a in args[:5]]
    kept = _run(hb, *eager, args[5])  # an eager graph that lives through the capture
    leaves = [a.clone().requires_grad_() for a in args[:5]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(sum(v.float().sum() for v in _run(hb, *leaves, args[5])), leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(hb, *leaves, args[5])
        grads = torch.autograd.grad(sum(v.float().sum() for v in out), leaves)
    gen = torch.Generator(device=cuda).manual_seed(2)
    for _ in range(3):
        with torch.no_grad():
            leaves[0].normal_(generator=gen)
        graph.replay()
        torch.cuda.synchronize()
        again = [v.detach().clone().requires_grad_() for v in leaves]
        want = _run(hb, *again, args[5])
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(sum(v.float().sum() for v in want), again)))
    sum(v.float().sum() for v in kept).backward()
    assert all(bool(torch.isfinite(v.grad).all()) for v in eager)


def test_two_threads(hb, cuda):
    """Calls of two host threads, each on a stream of its own, share nothing."""
    jobs = [_layer(hb, cuda, rows, dtype, rows) for rows, dtype in ((40, torch.float32), (700, torch.bfloat16))]
    want = [_run(hb, *job) for job in jobs]
    torch.cuda.synchronize()
    failed = []

    def work(job, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(60):
                got = _run(hb, *job)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    failed.append(len(job[0]))
                    return

    threads = [threading.Thread(target=work, args=pair) for pair in zip(jobs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_first_call_of_a_thread(hb, cuda):
    """A thread that has not used the device before, as autograd's may be: every call finds it."""
    x, gain, gate, up, down, first = _layer(hb, cuda, 400)
    dy = torch.ones((400, 128), dtype=torch.bfloat16, device=cuda)
    state = hb.adamw_state([gain.clone()], bits=8)
    torch.cuda.synchronize()
    calls = (lambda: hb.expert_product(x, gate, first), lambda: hb.expert_gated_grad(dy, x, gate, up, first), lambda: hb.rms_norm(x, gain),
             lambda: hb.expert_product_grad(dy, x, gate, first), lambda: hb.rms_norm_grad(x, x, gain),
             lambda: hb.adamw_step([gain.clone()], [gain], state, lr=0.1))
    failed = []

    def work(call):
        try:
            call()
        except Exception as e:  # noqa: BLE001
            failed.append(repr(e))

    for call in calls:
        t = threading.Thread(target=work, args=(call,))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed


def test_tangents_and_traces(hb, cuda):
    """Forward mode is refused, nothing is dropped silently; a trace holds the calls that have an autograd function."""
    x, gain, gate, up, down, first = _layer(hb, cuda, 40, torch.float32)
    dy = torch.ones((40, 128), device=cuda)
    state = hb.adamw_state([gain])
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: hb.expert_product(dual, gate, first), lambda: hb.expert_gated(dual, gate, up, first), lambda: hb.rms_norm(dual, gain),
                     lambda: hb.rms_norm_8bit(dual, gain), lambda: hb.rms_norm_grad(dual, x, gain), lambda: hb.expert_product_grad(dy, dual, gate, first),
                     lambda: hb.expert_gated_grad(dy, dual, gate, up, first), lambda: hb.adamw_step([x], [dual], hb.adamw_state([x]), lr=0.1)):
            with pytest.raises(NotImplementedError):
                call()
    traced = torch.jit.trace(lambda *a: _run(hb, *a), (x, gain, gate, up, down, first), check_trace=False)
    other = _layer(hb, cuda, 50, torch.float32, 9)
    assert all(torch.equal(a, b) for a, b in zip(traced(*other), _run(hb, *other)))
    for call in (lambda v: hb.rms_norm_8bit(v, gain)[0].scales, lambda v: hb.rms_norm_grad(v, x, gain)[0], lambda v: hb.expert_product_grad(dy, v, gate, first)[0],
                 lambda v: hb.expert_gated_grad(dy, v, gate, up, first)[0]):
        with pytest.raises(NotImplementedError, match="trace"):
            torch.jit.trace(call, (x,), check_trace=False)
    with pytest.raises(ValueError, match="number"):
        hb.adamw_step([gain], [gain.clone()], state, lr=torch.ones((), device=cuda, requires_grad=True))
    with pytest.raises(ValueError, match="number"):
        hb.rms_norm(x, gain, eps=torch.ones((), requires_grad=True))


def test_lazy_views(hb, cuda):
    """Lazily negated views and zeros without memory are read as what they stand for, or refused where they are written."""
    x, gain, gate, up, down, first = _layer(hb, cuda, 40, torch.float32)
    neg = torch.view_as_complex(torch.stack([torch.zeros_like(x), -x], -1)).conj().imag
    assert neg.is_neg() and torch.equal(neg, x)
    for got, want in ((hb.rms_norm(neg, gain), hb.rms_norm(x, gain)), (hb.expert_gated(neg, gate, up, first), hb.expert_gated(x, gate, up, first)),
                      (hb.expert_product_grad(torch.ones((40, 128), device=cuda), neg, gate, first)[1],
                       hb.expert_product_grad(torch.ones((40, 128), device=cuda), x, gate, first)[1])):
        assert torch.equal(got, want)
    zeros = torch._efficientzerotensor((40, 64), device=cuda)
    assert not hb.expert_product(zeros, gate, first).any() and not hb.rms_norm(zeros, gain).any()
    with pytest.raises(ValueError, match="memory"):
        hb.adamw_step([x], [neg], hb.adamw_state([x]), lr=0.1)


def test_beyond_32_bits(hb, cuda):
    """More than 2^31 elements: the last rows' values are those of the rows alone."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    rows, width = 1_100_000, 2048
    x = torch.empty((rows, width), dtype=torch.bfloat16, device=cuda)
    x[-300:] = torch.randn((300, width), generator=gen, device=cuda).to(torch.bfloat16)
    x[:-300].fill_(0.5)
    gain = torch.randn(width, generator=gen, device=cuda).to(torch.bfloat16)
    w = (torch.randn((2, 32, width), generator=gen, device=cuda) / 45).to(torch.bfloat16)
    first = torch.tensor([0, rows - 300, rows], dtype=torch.int32, device=cuda)
    tail = torch.tensor([0, 0, 300], dtype=torch.int32, device=cuda)
    assert torch.equal(hb.expert_product(x, w, first)[-300:], hb.expert_product(x[-300:], w, tail))
    assert torch.equal(hb.rms_norm(x, gain)[-300:], hb.rms_norm(x[-300:], gain))
    got, want = hb.rms_norm_8bit(x, gain)[0], hb.rms_norm_8bit(x[-300:], gain)[0]
    assert torch.equal(hb.rows_of_8bit(got, dtype=torch.bfloat16)[-300:], hb.rows_of_8bit(want, dtype=torch.bfloat16))
    dx, _ = hb.rms_norm_grad(x, x, gain)
    assert torch.equal(dx[-300:], hb.rms_norm_grad(x[-300:], x[-300:], gain)[0])
    del got, dx
    dy = torch.zeros((rows, 32), dtype=torch.bfloat16, device=cuda)
    dy[-300:] = torch.randn((300, 32), generator=gen, device=cuda).to(torch.bfloat16)
    dx, dw = hb.expert_product_grad(dy, x, w, first)
    dx2, dw2 = hb.expert_product_grad(dy[-300:], x[-300:], w, tail)
    assert torch.equal(dx[-300:], dx2) and not dx[:-300].any() and not dw[0].any()
    bound = 2 * 300 * E23 * float((dy[-300:].double().abs().t() @ x[-300:].double().abs()).max()) + 2 * ref.U[torch.bfloat16] * float(dw2.abs().max())
    assert float((dw[1] - dw2[1]).abs().max()) <= bound  # their parts may be cut elsewhere
    del dx, dx2, dy
    flat, grad = x.view(-1), torch.empty(rows * width, dtype=torch.bfloat16, device=cuda)
    grad.fill_(0.25)
    grad[-700:] = torch.randn(700, generator=gen, device=cuda).to(torch.bfloat16)
    piece = flat[-3 * 256:].clone()
    state = hb.adamw_state([flat], bits=8)
    hb.adamw_step([flat], [grad], state, lr=0.1)
    alone = hb.adamw_state([piece], bits=8)
    hb.adamw_step([piece], [grad[-3 * 256:].clone()], alone, lr=0.1)
    assert torch.equal(flat[-3 * 256:], piece)
    for a, b in ((state.exp_avg[0], alone.exp_avg[0]), (state.exp_avg_sq[0], alone.exp_avg_sq[0])):
        assert torch.equal(a[-3 * 256:].view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(state.exp_avg_scale[0][-3:], alone.exp_avg_scale[0])


def test_changed_before_backward(hb, cuda):
    """What the gradients need is saved as for any autograd function: written to in between, it is refused."""
    args = _layer(hb, cuda, 40, torch.float32)
    for place in (0, 2, 5):
        inputs = [a.clone() for a in args]
        gate = inputs[2].requires_grad_() if place != 2 else inputs[2]
        x = inputs[0].requires_grad_() if place == 2 else inputs[0]
        h = hb.expert_gated(x, gate, inputs[3], inputs[5])
        with torch.no_grad():
            inputs[place].add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            h.sum().backward()
