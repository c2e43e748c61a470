"""Routing by expert against plain 64-bit forms: the plan exactly, the moves exactly, the sums within
the fp32 summation bound (tests/rows_reference.py)."""
import numpy as np
import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu


def _index(rng, tokens, slots, experts, dropped, dtype=np.int64):
    index = rng.integers(0, experts, (tokens, slots)).astype(dtype)
    index[rng.random((tokens, slots)) < dropped] = rng.choice([-1, experts, experts + 7])
    return index


def _check_plan(plan, index, experts):
    order, position, offsets = ref.plan(index, experts)
    assert np.array_equal(plan.order.cpu().numpy(), order)
    assert np.array_equal(plan.position.cpu().numpy(), position)
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)


@pytest.mark.parametrize("tokens,slots,experts", [
    (1, 1, 1), (1, 2, 16), (31, 1, 2), (33, 3, 5), (511, 8, 64), (512, 8, 255), (513, 8, 256),  # one block, one pass
    (4096, 1, 2047), (4096, 1, 2048), (1365, 3, 70000), (1365, 3, 5_000_000),                   # two and three passes
    (4097, 1, 7), (5000, 3, 1024), (100, 100, 2047), (8193, 2, 300), (65537, 1, 5), (131072, 1, 2047),  # clusters
    (4097, 1, 2048), (20000, 2, 100003), (3000, 4, 5_000_000), (65536, 2, 65536),
    (131073, 1, 1024), (200000, 2, 100003), (140000, 1, 5_000_000),                             # tiles of 1024
    (2 ** 19 + 5, 1, 37), (70001, 8, 1025), (2 ** 19 + 1, 1, 4000), (2 ** 18 + 3, 2, 200), (2 ** 19, 1, 300)])                            # tiles of 4096
@pytest.mark.parametrize("dropped", [0.0, 0.2])
def test_plan_matches_counting(hb, cuda, tokens, slots, experts, dropped):
    rng = np.random.default_rng(tokens + slots)
    dtype = np.int32 if tokens % 2 else np.int64
    index = _index(rng, tokens, slots, experts, dropped, dtype)
    _check_plan(hb.route_plan(torch.as_tensor(index, device=cuda), experts), index, experts)


def test_plan_edges(hb, cuda):
    for n in (1, 40, 5000):  # no entry has an expert; one expert has all
        _check_plan(hb.route_plan(torch.full((n, 2), -1, device=cuda), 4), np.full((n, 2), -1), 4)
        _check_plan(hb.route_plan(torch.full((n, 2), 3, device=cuda), 4), np.full((n, 2), 3), 4)
    lows = np.array([np.iinfo(np.int64).min, np.iinfo(np.int64).max, 2 ** 32, 2 ** 32 + 1, -2 ** 32, 1, 0])
    _check_plan(hb.route_plan(torch.as_tensor(lows, device=cuda), 2), lows.reshape(-1, 1), 2)
    empty = hb.route_plan(torch.empty((0, 3), dtype=torch.int64, device=cuda), 5)
    assert empty.order.numel() == 0 and empty.position.shape == (0, 3) and empty.offsets.tolist() == [0] * 6
    assert hb.route_dispatch(torch.empty((0, 8), device=cuda), empty).shape == (0, 8)
    assert hb.route_combine(torch.empty((0, 8), device=cuda), empty).shape == (0, 8)
    strided = torch.as_tensor(np.arange(60).reshape(10, 6) % 7, device=cuda)[:, ::2]
    _check_plan(hb.route_plan(strided, 7), strided.cpu().numpy(), 7)
    plan = hb.route_plan(torch.tensor([2, 0, 2], device=cuda), 3)
    assert (plan.tokens, plan.slots, plan.num_experts, plan.counts.tolist()) == (3, 1, 3, [1, 0, 2])


CASES = [  # tokens, slots, experts, width, dropped
    (1, 2, 16, 2048, 0.0), (1, 1, 1, 1, 0.0), (5, 3, 4, 7, 0.3), (37, 3, 11, 1000, 0.2), (130, 5, 8, 257, 0.1),
    (1400, 3, 6, 1024, 0.1), (1300, 1, 6, 2048, 0.0), (1250, 2, 6, 1032, 0.1), (5000, 3, 9, 264, 0.1), (5000, 2, 9, 301, 0.1),
    (64, 9, 3, 40, 0.5), (2000, 2, 16, 128, 0.1), (1300, 4, 5, 516, 0.1), (3, 40, 64, 4104, 0.1), (17, 1, 4, 9000, 0.0)]


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("tokens,slots,experts,width,dropped", CASES)
def test_moves_match_64_bits(hb, cuda, dtype, tokens, slots, experts, width, dropped):
    rng = np.random.default_rng(tokens * 7 + width)
    index = _index(rng, tokens, slots, experts, dropped)
    plan = hb.route_plan(torch.as_tensor(index, device=cuda), experts)
    order, position, offsets = ref.plan(index, experts)
    kept = int(offsets[-1])

    def data(*shape):
        return torch.as_tensor(rng.normal(size=shape), device=cuda).to(dtype)

    x, z, dy = data(tokens, width), data(tokens * slots, width), data(tokens, width)
    weights = torch.as_tensor(rng.random((tokens, slots)), device=cuda).to(
        torch.float32 if tokens % 2 else dtype)
    z[kept:] = float("nan")  # rows without an expert are not read, nor their weights
    weights.view(-1)[torch.as_tensor(order[kept:], device=cuda)] = float("nan")
    x64, z64, dy64, w64 = ref.f64(x), ref.f64(z), ref.f64(dy), ref.f64(weights)

    want = np.zeros((tokens * slots, width))
    want[:kept] = x64[order[:kept] // slots]
    assert np.array_equal(ref.f64(hb.route_dispatch(x, plan)), want)

    u, floor = ref.U[dtype], ref.FLOOR[dtype]
    for w in (weights, None):
        want, mag = ref.combine(z64, position, kept, None if w is None else w64)
        ref.assert_within(hb.route_combine(z, plan, w), want,
                          slots * ref.E32 * mag * (1 + u) + u * np.abs(want) + floor, "combine")
    want, mag = ref.combine(z64, position, kept, None)
    ref.assert_within(hb.route_dispatch_grad(z, plan), want,
                      slots * ref.E32 * mag * (1 + u) + u * np.abs(want) + floor, "dispatch grad")

    live = order[:kept]
    dz, dw = hb.route_combine_grad(dy, z, plan, weights)
    want = np.zeros((tokens * slots, width))
    want[:kept] = dy64[live // slots] * w64.reshape(-1)[live][:, None]
    ref.assert_within(dz, want, (ref.E32 * (1 + u) + u) * np.abs(want) + floor, "dz")
    want, mag = np.zeros(tokens * slots), np.zeros(tokens * slots)
    want[live] = (dy64[live // slots] * z64[:kept]).sum(1)
    mag[live] = np.abs(dy64[live // slots] * z64[:kept]).sum(1)
    uw = ref.U[weights.dtype]
    ref.assert_within(dw.reshape(-1), want, width * ref.E32 * mag * (1 + uw) + uw * np.abs(want) + ref.FLOOR[weights.dtype],
                      "dw")
    dz1, none = hb.route_combine_grad(dy, z, plan)
    assert none is None
    want = np.zeros((tokens * slots, width))
    want[:kept] = dy64[live // slots]
    assert np.array_equal(ref.f64(dz1), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_addresses(hb, cuda, dtype):
    """Rows of a wider array, rows off the 16-byte grid, a transposed array and one row for all tokens."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    index = torch.randint(-1, 6, (50, 2), generator=gen, device=cuda)
    plan = hb.route_plan(index, 6)
    wide = torch.randn((100, 300), generator=gen, device=cuda).to(dtype)
    for z in (wide[:, :256], wide[:, 1:258], wide[:, 3:11], wide[:, 2:4], wide.t().contiguous().t()[:, :200]):
        x = z[:50]
        assert torch.equal(hb.route_dispatch(x, plan), hb.route_dispatch(x.contiguous(), plan))
        w = torch.rand((2, 50), generator=gen, device=cuda).t()
        assert torch.equal(hb.route_combine(z, plan, w), hb.route_combine(z.contiguous(), plan, w.contiguous()))
        dz, dw = hb.route_combine_grad(x, z, plan, w)
        assert torch.equal(dz, hb.route_combine_grad(x.contiguous(), z.contiguous(), plan, w)[0])
        # dw's order of summation goes by the vectors that the addresses allow: against 64 bits instead
        live = (plan.position < plan.offsets[-1]).double()
        pairs = x.double().unsqueeze(1) * z.double()[plan.position.long()]
        assert bool(((dw.double() - live * pairs.sum(2)).abs() <= z.shape[1] * ref.E32 * pairs.abs().sum(2)).all())
    one = wide[:1, :64].expand(50, 64)
    assert torch.equal(hb.route_dispatch(one, plan), hb.route_dispatch(one.contiguous(), plan))


def test_autograd_and_differences(hb, cuda):
    """The layer combine(tanh(dispatch(x)), w): gradients through autograd equal the formulas', and the change
    of the loss along a direction (central differences in 64 bits of the fp32 outputs)."""
    rng = np.random.default_rng(3)
    tokens, slots, experts, width = 40, 2, 5, 24
    index = _index(rng, tokens, slots, experts, 0.1)
    plan = hb.route_plan(torch.as_tensor(index, device=cuda), experts)
    order, position, offsets = ref.plan(index, experts)
    kept = int(offsets[-1])
    x = torch.as_tensor(rng.normal(size=(tokens, width)), dtype=torch.float32, device=cuda).requires_grad_()
    w = torch.as_tensor(rng.random((tokens, slots)), dtype=torch.float32, device=cuda).requires_grad_()
    r = torch.as_tensor(rng.normal(size=(tokens, width)), dtype=torch.float32, device=cuda)

    def loss64(xv, wv):  # the formula in 64 bits
        z = np.zeros((tokens * slots, width))
        z[:kept] = np.tanh(xv[order[:kept] // slots])
        return float((ref.combine(z, position, kept, wv)[0] * ref.f64(r)).sum())

    y = hb.route_combine(torch.tanh(hb.route_dispatch(x, plan)), plan, w)
    (y * r).sum().backward()
    x64, w64 = ref.f64(x), ref.f64(w)
    assert abs(float((y.detach().double() * r.double()).sum()) - loss64(x64, w64)) < 1e-3
    h = 1e-5
    for grad, at in ((x.grad, 0), (w.grad, 1)):
        for _ in range(4):
            v = rng.normal(size=grad.shape)
            move = [(x64 + s * h * v, w64) if at == 0 else (x64, w64 + s * h * v) for s in (1, -1)]
            change = (loss64(*move[0]) - loss64(*move[1])) / (2 * h)
            # fp32 gradients: about 2^-22 of the summed magnitudes; differences: h^2 and 2^-53 / h
            assert abs(float((ref.f64(grad) * v).sum()) - change) <= 2.0 ** -18 * np.abs(ref.f64(grad) * v).sum() + 1e-7


def test_autograd_without_weights(hb, cuda):
    index = torch.tensor([[0, 1], [1, -1], [0, 0]], device=cuda)
    plan = hb.route_plan(index, 2)
    z = torch.randn((6, 5), device=cuda).requires_grad_()
    hb.route_combine(z, plan).sum().backward()
    assert torch.equal(z.grad, torch.tensor([1.0, 1, 1, 1, 1, 0], device=cuda).unsqueeze(1).expand(6, 5))


def test_lazily_negated_rows(hb, cuda):
    """The imaginary part of a conjugate is a view whose memory has the other sign."""
    rows = torch.randn((4, 3), dtype=torch.complex64, device=cuda).conj().imag
    assert rows.is_neg()
    plan = hb.route_plan(torch.tensor([1, 0, 1, 0], device=cuda), 2)
    assert torch.equal(hb.route_dispatch(rows, plan), rows.resolve_neg()[plan.order.long()])


def test_other_stream_and_graph(hb, cuda):
    """Work goes to the current stream, and a captured step replays on new data."""
    gen = torch.Generator(device=cuda).manual_seed(5)
    x = torch.randn((3000, 64), generator=gen, device=cuda)
    index = torch.randint(0, 9, (3000, 2), generator=gen, device=cuda)
    w = torch.rand((3000, 2), generator=gen, device=cuda)

    def step():
        plan = hb.route_plan(index, 9)
        return hb.route_combine(hb.route_dispatch(x, plan), plan, w)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.normal_(generator=gen)
    index.random_(0, 9, generator=gen)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, step())


def test_more_than_2_31_elements(hb, cuda):
    """Rows beyond element 2^31 of the sorted array arrive and come back."""
    tokens, slots, width = 140_000, 8, 2048
    assert tokens * slots * width > 2 ** 31
    index = torch.arange(tokens * slots, device=cuda).view(tokens, slots) % 11
    plan = hb.route_plan(index, 11)
    x = (torch.arange(tokens, device=cuda) % 251).to(torch.bfloat16).unsqueeze(1).expand(tokens, width)
    rows = hb.route_dispatch(x, plan)
    back = hb.route_combine(rows, plan)
    assert torch.equal(rows[:, 5], x[(plan.order // slots).long(), 0])
    assert torch.equal(rows[-1], x[int(plan.order[-1]) // slots])
    assert torch.equal(back[:, 2047], (x[:, 0].float() * slots).to(torch.bfloat16))


def test_refusals(hb, cuda):
    index = torch.zeros((4, 2), dtype=torch.int64, device=cuda)
    for bad in (index.float(), index.view(1, 4, 2), index.cpu(), torch.empty((4, 0), dtype=torch.int64, device=cuda)):
        with pytest.raises(ValueError):
            hb.route_plan(bad, 3)
    for experts in (0, -1, 2 ** 31):
        with pytest.raises(ValueError):
            hb.route_plan(index, experts)
    plan = hb.route_plan(index, 3)
    x, z, w = (torch.zeros(s, device=cuda) for s in ((4, 6), (8, 6), (4, 2)))
    for call in (lambda: hb.route_dispatch(x[:3], plan), lambda: hb.route_dispatch(x.double(), plan),
                 lambda: hb.route_dispatch(x.cpu(), plan), lambda: hb.route_dispatch(x[0], plan),
                 lambda: hb.route_dispatch(x, plan._replace(position=plan.position.long())),
                 lambda: hb.route_dispatch(x, plan._replace(position=plan.position.view(-1))),
                 lambda: hb.route_combine(x, plan), lambda: hb.route_combine(z, plan, w[:3]),
                 lambda: hb.route_combine(z, plan, w.long()), lambda: hb.route_combine(z, plan, w.cpu()),
                 lambda: hb.route_combine_grad(x.half(), z, plan, w), lambda: hb.route_combine_grad(z, z, plan, w)):
        with pytest.raises(ValueError):
            call()


def test_assignment_of_a_transport_plan(hb, cuda):
    rows, cols = np.array([2, 0, 0, 2, 1, 2]), np.array([4, 1, 3, 0, 2, 1])
    mass = np.array([0.25, 0.1, 0.4, 0.25, 0.0, 0.5])
    index, weights = hb.assignment_of_plan(rows, cols, mass, 4, device=cuda)
    assert index.tolist() == [[3, 1, -1], [-1, -1, -1], [1, 0, 4], [-1, -1, -1]]
    assert np.allclose(weights.cpu().numpy(), [[0.8, 0.2, 0], [0, 0, 0], [0.5, 0.25, 0.25], [0, 0, 0]], atol=1e-7)
