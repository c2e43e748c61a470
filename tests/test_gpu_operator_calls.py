"""What the routing, lookup and clipping calls keep to beside their results on ordinary arguments."""
import threading
import time

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fw

import rows_reference as ref

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


def test_forward_mode_of_the_linear_calls(hb, cuda):
    """Dispatch and lookup are linear: the tangent goes the values' way, bit for bit, with or without grad mode."""
    gen = torch.Generator(device=cuda).manual_seed(2)
    plan = _plan(hb, cuda, gen)
    ids = torch.randint(-1, 40, (3, 7), generator=gen, device=cuda)
    for dtype in ref.DTYPES:
        x, t = (torch.randn((40, 24), generator=gen, device=cuda).to(dtype) for _ in range(2))
        for call in (lambda v: hb.route_dispatch(v, plan), lambda v: hb.embedding_lookup(v, ids, scale=1.5)):
            for mode in (True, False):
                with torch.set_grad_enabled(mode), fw.dual_level():
                    value, tangent = fw.unpack_dual(call(fw.make_dual(x, t)))
                    assert torch.equal(value, call(x)) and torch.equal(tangent, call(t))


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_forward_mode_of_combine(hb, cuda, dtype):
    """The tangent of sum w z is sum (w dz + dw z), 2 slots products in fp32 rounded once."""
    rng = np.random.default_rng(3)
    gen = torch.Generator(device=cuda).manual_seed(3)
    tokens, slots, width = 40, 3, 24
    plan = _plan(hb, cuda, gen, tokens, slots)
    position, kept = plan.position.cpu().numpy(), int(plan.offsets[-1])
    z, dz = (torch.as_tensor(rng.normal(size=(tokens * slots, width)), device=cuda).to(dtype) for _ in range(2))
    w, dw = (torch.as_tensor(rng.random((tokens, slots)), device=cuda).to(dtype) for _ in range(2))
    u, floor = ref.U[dtype], ref.FLOOR[dtype]
    for with_z, with_w in ((True, False), (False, True), (True, True)):
        want, mag = np.zeros((tokens, width)), np.zeros((tokens, width))
        for on, rows, weights in ((with_z, dz, w), (with_w, z, dw)):
            if on:
                part = ref.combine(ref.f64(rows), position, kept, ref.f64(weights))
                want, mag = want + part[0], mag + part[1]
        with fw.dual_level():
            value, tangent = fw.unpack_dual(hb.route_combine(fw.make_dual(z, dz) if with_z else z, plan,
                                                             fw.make_dual(w, dw) if with_w else w))
        assert torch.equal(value, hb.route_combine(z, plan, w))
        ref.assert_within(tangent, want, 2 * slots * ref.E32 * mag * (1 + u) + u * np.abs(want) + floor)
    with fw.dual_level():
        tangent = fw.unpack_dual(hb.route_combine(fw.make_dual(z, dz), plan)).tangent
    assert torch.equal(tangent, hb.route_combine(dz, plan))
    # a derivative along z of the derivative along w, whose graph goes through the tangent
    z = z.clone().requires_grad_()
    with fw.dual_level():
        fw.unpack_dual(hb.route_combine(z, plan, fw.make_dual(w, dw))).tangent.sum().backward()
    assert torch.equal(z.grad, hb.route_combine_grad(torch.ones((tokens, width), dtype=dtype, device=cuda), z.detach(),
                                                     plan, dw)[0])


def test_tangents_are_not_dropped(hb, cuda):
    """Calls without a derivative of their own refuse a tensor that carries a tangent."""
    gen = torch.Generator(device=cuda).manual_seed(4)
    plan = _plan(hb, cuda, gen)
    ids = torch.randint(0, 9, (40,), generator=gen, device=cuda)
    x, z, w = (torch.randn(s, generator=gen, device=cuda) for s in ((40, 8), (80, 8), (40, 2)))
    with fw.dual_level():
        dx, dz, dw = (fw.make_dual(v, torch.ones_like(v)) for v in (x, z, w))
        for call in (lambda: hb.route_dispatch_grad(dz, plan), lambda: hb.route_combine_grad(dx, z, plan, w),
                     lambda: hb.route_combine_grad(x, dz, plan, w), lambda: hb.route_combine_grad(x, z, plan, dw),
                     lambda: hb.embedding_grad(dx, ids, 9), lambda: hb.grad_norm([x, dx]),
                     lambda: hb.clip_grad_norm([dx], 1.0), lambda: hb.clip_grad_norm([x], 1.0, out=[dx])):
            with pytest.raises(NotImplementedError, match="tangent"):
                call()


def test_zeros_without_memory(hb, cuda):
    """Tangents can be zeros that have no memory, rows and weights alike."""
    gen = torch.Generator(device=cuda).manual_seed(7)
    plan = _plan(hb, cuda, gen)
    z, w = torch.randn((80, 8), generator=gen, device=cuda), torch.rand((40, 2), generator=gen, device=cuda)
    none = {shape: torch._efficientzerotensor(shape, device=cuda) for shape in ((40, 8), (80, 8), (40, 2))}
    for got in (hb.route_dispatch(none[40, 8], plan), hb.route_combine(none[80, 8], plan, w),
                hb.route_combine(z, plan, none[40, 2]), hb.embedding_lookup(none[40, 8], torch.arange(5, device=cuda))):
        assert not got._is_zerotensor() and not got.any()


def _traced(call, *inputs):
    return torch.jit.trace(call, inputs, check_trace=False)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("grad", [False, True])
def test_traced_calls_run_again(hb, cuda, grad):
    """A trace holds the call itself, on new rows and on a new plan."""
    gen = torch.Generator(device=cuda).manual_seed(5)

    def inputs():
        x, z = (torch.randn(s, generator=gen, device=cuda).requires_grad_(grad) for s in ((40, 8), (80, 8)))
        w, ids = torch.rand((40, 2), generator=gen, device=cuda), torch.randint(0, 40, (6,), generator=gen, device=cuda)
        plan = _plan(hb, cuda, gen)
        return x, z, w, ids, plan.order, plan.position, plan.offsets

    def layer(x, z, w, ids, order, position, offsets):
        plan = hb.RoutePlan(order, position, offsets)
        return (hb.route_dispatch(x, plan), hb.route_combine(z, plan, w), hb.route_combine(z, plan),
                hb.embedding_lookup(x, ids, scale=2.0))

    traced = _traced(layer, *inputs())
    other = inputs()
    for got, want in zip(traced(*other), layer(*other)):
        assert torch.equal(got, want)


@pytest.mark.filterwarnings("ignore")
def test_calls_that_a_trace_cannot_hold(hb, cuda):
    gen = torch.Generator(device=cuda).manual_seed(6)
    plan = _plan(hb, cuda, gen)
    x, z = (torch.randn(s, generator=gen, device=cuda) for s in ((40, 8), (80, 8)))
    ids = torch.zeros(40, dtype=torch.int64, device=cuda)
    for call, at in ((lambda v: hb.route_plan(v, 3).order, ids), (lambda v: hb.route_dispatch_grad(v, plan), z),
                     (lambda v: hb.route_combine_grad(v, z, plan)[0], x), (lambda v: hb.embedding_grad(v, ids, 4), x),
                     (lambda v: hb.grad_norm([v]), x), (lambda v: hb.clip_grad_norm([v], 1.0), x)):
        with pytest.raises(NotImplementedError, match="trace"):
            _traced(call, at)


def test_numbers_carry_no_gradient(hb, cuda):
    table, ids = torch.ones((4, 3), device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
    scale = torch.tensor(2.0, requires_grad=True)
    assert torch.equal(hb.embedding_lookup(table, ids, scale=scale.detach()), 2 * table[:2])
    with torch.no_grad():
        hb.embedding_lookup(table, ids, scale=scale)
    for call in (lambda: hb.embedding_lookup(table, ids, scale=scale), lambda: hb.embedding_grad(table[:2], ids, 4, scale=scale),
                 lambda: hb.embedding_lookup(table.clone().requires_grad_(), ids, scale=scale),
                 lambda: hb.clip_grad_norm([table], scale)):
        with pytest.raises(ValueError, match="number"):
            call()


def test_clipping_needs_a_limit(hb, cuda):
    g = torch.full((4,), 3.0, device=cuda)
    out = torch.full_like(g, 7.0)
    for kwargs in ({}, {"out": [out]}):
        with pytest.raises((TypeError, ValueError)):
            hb.clip_grad_norm([g], None, **kwargs)


def test_lookup_of_an_empty_table_has_a_gradient(hb, cuda):
    table = torch.empty((0, 8), device=cuda).requires_grad_()
    y = hb.embedding_lookup(table, torch.tensor([0, -1, 3], device=cuda))
    assert y.shape == (3, 8) and not y.any()
    y.sum().backward()
    assert table.grad.shape == (0, 8)


def test_clipping_refuses_shared_memory(hb, cuda):
    """Outputs that overlap one another, or a gradient that is not their own, would be written while they are read."""
    flat = torch.arange(1.0, 65.0, device=cuda)
    a, b = flat[:16], flat[16:32]
    half = torch.ones(32, dtype=torch.bfloat16, device=cuda)
    kept = flat.clone()
    for grads, out in (([a, b], [b, a]), ([a, b], [torch.empty_like(a), a]), ([flat, flat[10:20]], None), ([flat[10:20], flat], None),
                       ([a, b], [flat[1:17], flat[32:48]]), ([a], [flat[15:31]]), ([b], [flat[1:17]]),
                       ([kept[:16], kept[16:32]], [flat[:16], flat[15:31]]), ([half[:16]], [half.view(torch.float32)[:16]]),
                       ([half[:8], half[8:16]], [torch.empty(8, device=cuda), half.view(torch.float32)[:8]])):
        with pytest.raises(ValueError, match="overlap|in place"):
            hb.clip_grad_norm(grads, 1.0, out=out)
    assert torch.equal(flat, kept) and bool((half == 1).all())


def test_clipping_takes_neighbours_in_memory(hb, cuda):
    """Slices of one buffer, in place and beside it; gradients that are only read may overlap."""
    flat = torch.arange(1.0, 65.0, device=cuda)
    norm = hb.grad_norm([flat[:20], flat[10:30]])
    want = torch.cat([flat[:20], flat[10:30]]).double().norm()
    assert abs(float(norm) - float(want)) <= 17 * ref.E32 * float(want)
    out = torch.empty(40, device=cuda)
    assert torch.equal(hb.clip_grad_norm([flat[:20], flat[10:30]], 1.0, out=[out[20:], out[:20]]), norm)
    factor = 1.0 / (float(want) + 1e-6)
    for got, g in ((out[20:], flat[:20]), (out[:20], flat[10:30])):
        assert bool(((got.double() - g.double() * factor).abs() <= 21 * ref.E32 * g.double() * factor).all())
    both = flat.clone()
    hb.clip_grad_norm([both[:10], both[10:64]], 1.0, out=[both[:10], both[10:64]])
    alone = flat.clone()
    hb.clip_grad_norm([alone[:10], alone[10:64]], 1.0)
    assert torch.equal(both, alone) and not torch.equal(both, flat)
    empty = flat[5:5]
    hb.clip_grad_norm([alone, empty], 1.0, out=[both, empty])


def test_table_gradient_refuses_to_write_its_rows(hb, cuda):
    """out is written while dy is read: they may lie in one buffer, between rows too, but share nothing."""
    gen = torch.Generator(device=cuda).manual_seed(8)
    flat = torch.randn(400, generator=gen, device=cuda)
    kept = flat.clone()
    ids = torch.tensor([2, 0, 2, 1, -1], device=cuda)
    dy = flat[100:200].view(5, 20)[:, :8]  # rows of 8 at 100, 120, 140, 160, 180
    for start, rows in ((100, 5), (93, 1), (107, 1), (60, 6), (112, 2), (185, 3), (90, 20), (181, 1)):
        out = flat[start:start + rows * 8].view(rows, 8)
        for accumulate in (False, True):
            with pytest.raises(ValueError, match="overlap"):
                hb.embedding_grad(dy, ids, rows, out=out, accumulate=accumulate)
    with pytest.raises(ValueError, match="overlap"):
        hb.embedding_grad(flat[:8].expand(5, 8), ids, 3, out=flat[4:28].view(3, 8))
    assert torch.equal(flat, kept)
    for start, rows in ((76, 3), (188, 3), (108, 1), (112, 1), (170, 1)):
        out = flat[start:start + rows * 8].view(rows, 8)
        assert torch.equal(hb.embedding_grad(dy, ids, rows, out=out), hb.embedding_grad(kept[100:200].view(5, 20)[:, :8], ids, rows))
        flat.copy_(kept)
    t = flat[:40].view(8, 5).t()  # copied before it is read
    want = hb.embedding_grad(t.contiguous(), ids, 3)
    assert torch.equal(hb.embedding_grad(t, ids, 3, out=flat[:24].view(3, 8)), want)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("width", [64, 2, 1])
def test_accumulated_subnormals(hb, cuda, dtype, width):
    """Values below fp32's least normal number are added like any other, and a sum is rounded once: with rows of
    one token the result is scale * dy + out in 64 bits, rounded to fp32 at the end."""
    rng = np.random.default_rng(width)
    n, rows = 50, 60
    tiny = 2.0 ** -140
    scale = 0.75 if dtype == torch.float32 else 2.0 ** -130  # of fp16's range, products below it
    size = tiny if dtype == torch.float32 else 1.0
    dy = torch.as_tensor(rng.normal(size=(n, width)) * size, device=cuda).to(dtype)
    ids = torch.as_tensor(rng.permutation(rows)[:n], device=cuda)
    base = torch.as_tensor(rng.normal(size=(rows, width)) * tiny, device=cuda).to(torch.float32)
    out = base.clone()
    hb.embedding_grad(dy, ids, rows, scale=scale, out=out, accumulate=True)
    want = ref.f64(base)
    want[ids.cpu().numpy()] += ref.f64(dy) * scale
    assert np.array_equal(ref.f64(out), want.astype(np.float32).astype(np.float64))


def test_sorts_from_two_threads(hb, cuda):
    """The C entries share nothing between calls: two host threads sort by different numbers of bins, whose kernels
    differ in shared memory."""
    lib, n = hb.load_library(), 30_000
    gen = torch.Generator(device=cuda).manual_seed(9)
    failed = []

    def work(n, bins, stream):
        index = torch.randint(0, bins, (n,), generator=gen, device=cuda, dtype=torch.int32)
        order, position = (torch.empty(n, dtype=torch.int32, device=cuda) for _ in range(2))
        offsets = torch.empty(bins + 1, dtype=torch.int32, device=cuda)
        size = lib.hb_index_sort_workspace(n, bins)
        ws = torch.empty(max(size, 1), dtype=torch.uint8, device=cuda)
        torch.cuda.synchronize()

        def loop():
            for _ in range(400):
                rc = lib.hb_index_sort(index.data_ptr(), 4, n, bins, order.data_ptr(), position.data_ptr(),
                                       offsets.data_ptr(), ws.data_ptr(), size, stream.cuda_stream)
                if rc:
                    failed.append((bins, rc, lib.hb_last_error()))
                    return
        return loop, index, order

    for n in (30_000, 100_000):
        jobs = [work(n, bins, torch.cuda.Stream()) for bins in (2000, 900)]
        threads = [threading.Thread(target=job[0]) for job in jobs]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not failed, failed
        for _, index, order in jobs:
            assert torch.equal(order.long(), torch.sort(index, stable=True).indices)


@pytest.mark.parametrize("sizes", [[1 << 19], [8000 - i for i in range(64)], [100_000, 8192 * 20 + 5, 3], [8193] * 31])
def test_clipping_in_place_in_one_launch(hb, cuda, sizes):
    """More chunks than the cluster has blocks: in place the same values as beside, and those within the bounds."""
    gen = torch.Generator(device=cuda).manual_seed(len(sizes))
    for dtype in ref.DTYPES:
        grads = [torch.randn(n, generator=gen, device=cuda).to(dtype) for n in sizes]
        norm = float(torch.stack([g.double().square().sum() for g in grads]).sum().sqrt())
        out = [torch.empty_like(g) for g in grads]
        got = hb.clip_grad_norm(grads, 0.5 * norm, out=out)
        assert abs(float(got) - norm) <= 17 * ref.E32 * norm
        factor = 0.5 * norm / (norm + 1e-6)
        for g, o in zip(grads, out):
            want = ref.f64(g) * factor
            ref.assert_within(o, want, (20 * ref.E32 * (1 + ref.U[dtype]) + ref.U[dtype]) * np.abs(want) + ref.FLOOR[dtype])
        assert torch.equal(hb.clip_grad_norm(grads, 0.5 * norm), got)
        assert all(torch.equal(g, o) for g, o in zip(grads, out))


# ------------------------------------------------------------------ launches that overlap
@pytest.mark.parametrize("n,bins", [(1500, 9000), (30_000, 70), (30_000, 90_000), (200_000, 1024), (200_000, 100_003),
                                    (600_000, 37), (600_000, 5000)])
def test_captured_sorts(hb, cuda, n, bins):
    """Every form of the sort, captured and replayed on new entries back to back; a launch of the row may start while
    the one before ends."""
    gen = torch.Generator(device=cuda).manual_seed(n + bins)
    index = torch.empty(n, dtype=torch.int64, device=cuda)
    index.random_(-1, bins, generator=gen)
    hb.route_plan(index, bins)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = hb.route_plan(index, bins)
    for _ in range(20):
        index.random_(-1, bins, generator=gen)
        graph.replay()
        got = [t.clone() for t in plan]
        key = torch.where(index >= 0, index, bins)
        keys, order = torch.sort(key, stable=True)
        assert torch.equal(got[0].long(), order)
        assert torch.equal(got[1].view(-1)[order].long(), torch.arange(n, device=cuda))
        assert torch.equal(got[2].long(), torch.searchsorted(keys, torch.arange(bins + 1, device=cuda)))


@pytest.mark.parametrize("n,rows,width", [(1000, 5003, 129), (30_000, 700, 64), (150_000, 5000, 32), (150_000, 900, 9)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_captured_table_gradients(hb, cuda, n, rows, width, accumulate):
    """The gradient starts while its sort ends: captured and replayed on new tokens, equal to the call, bit for bit."""
    gen = torch.Generator(device=cuda).manual_seed(n)
    ids = torch.empty(n, dtype=torch.int32, device=cuda)
    dy = torch.empty((n, width), dtype=torch.bfloat16, device=cuda)
    out = torch.zeros((rows, width), device=cuda)

    def fill():
        ids.random_(-1, rows, generator=gen)
        dy.normal_(generator=gen)

    fill()
    hb.embedding_grad(dy, ids, rows, out=out, accumulate=accumulate)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hb.embedding_grad(dy, ids, rows, out=out, accumulate=accumulate)
    for _ in range(10):
        fill()
        want = out.clone()
        graph.replay()
        assert torch.equal(out, hb.embedding_grad(dy, ids, rows, out=want, accumulate=accumulate))


def test_two_streams_at_once(hb, cuda):
    """Calls with workspaces on two streams overlap and share nothing."""
    gen = torch.Generator(device=cuda).manual_seed(11)
    n, rows, width = 60_000, 3000, 96
    jobs = [(torch.randn((n, width), generator=gen, device=cuda), torch.randint(-1, rows, (n, 2), generator=gen, device=cuda),
             torch.randn(3_000_000, generator=gen, device=cuda)) for _ in range(2)]

    def work(x, index, g):
        plan = hb.route_plan(index, rows)
        y = hb.route_combine(hb.route_dispatch(x, plan), plan)
        out = torch.empty_like(g)
        norm = hb.clip_grad_norm([g], 1.0, out=[out])
        return [*plan, y, hb.embedding_grad(x, index[:, 0], rows), out, norm]

    want = [work(*job) for job in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(8):
        got = []
        for stream, job in zip(streams, jobs):
            with torch.cuda.stream(stream):
                got.append(work(*job))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_other_threads_go_on_while_the_launch_queue_is_full(hb, cuda):
    """A launch waits when the device is a thousand launches behind; other Python threads do not wait with it."""
    gen = torch.Generator(device=cuda).manual_seed(12)
    plan = _plan(hb, cuda, gen)
    x, z = torch.randn((40, 8), generator=gen, device=cuda), torch.randn((80, 8), generator=gen, device=cuda)
    ids = torch.zeros(40, dtype=torch.int64, device=cuda)
    calls = (lambda: hb.route_dispatch(x, plan), lambda: hb.route_combine(z, plan), lambda: hb.embedding_lookup(x, ids),
             lambda: hb.grad_norm([x]), lambda: hb.route_plan(ids, 3), lambda: hb.embedding_grad(x, ids, 3),
             lambda: hb.route_combine_grad(x, z, plan))
    for call in calls:
        call()
        torch.cuda.synchronize()
        seen, done = [], threading.Event()

        def watch():
            while not done.is_set():
                seen.append(time.perf_counter())
                time.sleep(0.002)

        watcher = threading.Thread(target=watch)
        watcher.start()
        torch.cuda._sleep(800_000_000)  # some 0.4 s
        start = time.perf_counter()
        for _ in range(2500):
            call()
        took = time.perf_counter() - start
        done.set()
        watcher.join()
        torch.cuda.synchronize()
        assert took > 0.2, "the queue was not full"
        longest = max(b - a for a, b in zip(seen, seen[1:]))
        assert longest < took / 2
