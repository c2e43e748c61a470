"""The experts' products against 64-bit forms (bounds: tests/expert_reference.py)."""
import pytest
import torch

import expert_reference as er
import rows_reference as ref

pytestmark = pytest.mark.gpu

# counts of each expert, rows behind the last, width, hidden: both tile forms, tiles' edges, empty experts, odd sizes
SHAPES = {
    "one row": ([1], 0, 64, 64),
    "few": ([0, 2, 1, 0, 5], 3, 72, 40),
    "few, odd": ([3, 0, 9], 0, 33, 17),
    "few, long": ([7, 9], 0, 2048, 130),
    "small experts": ([20, 1, 0, 127, 128, 129, 64], 11, 96, 136),
    "small experts, odd": ([33, 70, 2], 5, 61, 201),
    "large experts": ([300, 0, 513, 256], 40, 320, 264),
    "large experts, odd": ([400, 129, 300], 3, 131, 259),
    "large experts, long": ([700, 400], 0, 1096, 520),
    "dense": ([1100], 0, 200, 136),
    "many experts": ([i % 4 for i in range(700)], 2, 40, 24),
    "narrow": ([150, 90], 0, 1, 3),
}
GRADS = [k for k in SHAPES]


def _data(cuda, shape, dtype, seed=0):
    counts, behind, width, hidden = SHAPES[shape]
    gen = torch.Generator(device=cuda).manual_seed(seed + len(shape))
    offsets, rows = er.groups(counts, behind)

    def normal(*size, scale=1.0):
        return (torch.randn(size, generator=gen, device=cuda) * scale).to(dtype)

    x, dy = normal(rows, width), normal(rows, hidden)
    w = [normal(len(counts), hidden, width, scale=width ** -0.5) for _ in range(2)]
    x[offsets[-1]:], dy[offsets[-1]:] = float("nan"), float("inf")  # rows without an expert may hold anything
    return x, dy, w, offsets, torch.tensor(offsets, dtype=torch.int32, device=cuda)


def _live(v, offsets):
    v = v.double()
    v[offsets[-1]:] = 0
    return v


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(hb, cuda, shape, dtype):
    x, _, (gate, up), offsets, first = _data(cuda, shape, dtype)
    x64 = _live(x, offsets)
    y = hb.expert_product(x, gate, first)
    assert y.dtype == dtype and not y[offsets[-1]:].any()
    er.close(y, *er.product(x64, gate.double(), offsets, dtype), "product")
    for name in ("silu", "gelu"):
        h = hb.expert_gated(x, gate, up, first, activation=name)
        assert h.dtype == dtype and not h[offsets[-1]:].any()
        er.close(h, *er.gated(x64, gate.double(), up.double(), offsets, name, dtype), name)
    assert torch.equal(h, hb.expert_gated(x, gate, up, first, activation="gelu"))


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("shape", GRADS)
def test_gradients(hb, cuda, shape, dtype):
    x, dy, (gate, up), offsets, first = _data(cuda, shape, dtype)
    x64, dy64 = _live(x, offsets), _live(dy, offsets)
    got = hb.expert_product_grad(dy, x, gate, first)
    for name, g, (want, bound) in zip(("dx", "dw"), got, er.product_grad(dy64, x64, gate.double(), offsets, dtype)):
        assert g.dtype == dtype
        er.close(g, want, bound, name)
    for act in ("silu", "gelu"):
        got = hb.expert_gated_grad(dy, x, gate, up, first, activation=act)
        wants = er.gated_grad(dy64, x64, gate.double(), up.double(), offsets, act, dtype)
        for name, g, (want, bound) in zip(("dx", "dgate", "dup"), got, wants):
            assert g.dtype == dtype
            er.close(g, want, bound, f"{act} {name}")
    again = hb.expert_gated_grad(dy, x, gate, up, first, activation="gelu")
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for needs in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        part = hb.expert_gated_grad(dy, x, gate, up, first, activation="gelu", needs=needs)
        for need, p, (want, bound) in zip(needs, part, wants):
            assert (p is not None) == need
            if need:
                er.close(p, want, bound, needs)
    for needs in ((True, False), (False, True)):
        part = hb.expert_product_grad(dy, x, gate, first, needs=needs)
        assert [p is not None for p in part] == list(needs)


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_rows_do_not_reach_one_another(hb, cuda, dtype):
    """A row that is not finite reaches its own outputs and its expert's weight gradients, nothing else."""
    x, dy, (gate, up), offsets, first = _data(cuda, "small experts", dtype)
    bad = offsets[4] - 1  # the last row of the expert before a boundary inside a tile and a stage
    clean = [hb.expert_gated(x, gate, up, first), *hb.expert_gated_grad(dy, x, gate, up, first), *hb.expert_product_grad(dy, x, gate, first)]
    x[bad] = float("nan")
    dy[bad] = float("inf")
    got = [hb.expert_gated(x, gate, up, first), *hb.expert_gated_grad(dy, x, gate, up, first), *hb.expert_product_grad(dy, x, gate, first)]
    for c, g in zip(clean, got):
        keep = torch.ones(g.shape[0], dtype=torch.bool, device=cuda)
        keep[bad if g.dim() == 2 else 3] = False
        assert torch.equal(c[keep], g[keep]) and not bool(torch.isfinite(g[~keep]).all())


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("rows", [9, 300, 900, 5000])
def test_dense_and_strided(hb, cuda, dtype, rows):
    """Weights of one expert in two dimensions, halves of one weight, rows and weights off the 16-byte grid, other
    orders, expanded rows and weights: the values of dense copies."""
    gen = torch.Generator(device=cuda).manual_seed(rows)
    width, hidden = 88, 48

    def normal(*size):
        return torch.randn(size, generator=gen, device=cuda).to(dtype)

    both = normal(2, 2 * hidden, width)
    wide = normal(rows, width + 16)
    dy_wide = normal(rows, hidden + 3)
    flat = normal(rows * width + 1)
    off = normal(2 * hidden * width + 3)
    first = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device=cuda)
    for x in (wide[:, 8:width + 8], wide[:, 3:width + 3], flat[1:].view(rows, width), wide[:, :width].t().contiguous().t(),
              wide[:1, :width].expand(rows, width)):
        for gate, up in ((both[:, :hidden], both[:, hidden:]), (off[3:].view(2, hidden, width), both[:, :hidden]),
                         (both[:, ::2], both[:, 1::2]), (both[:1, :hidden].expand(2, hidden, width), both[:, :hidden])):
            plain = [v.contiguous().clone() for v in (x, gate, up)]
            wide64, offsets = [v.double() for v in plain], first.tolist()
            er.close(hb.expert_gated(x, gate, up, first), *er.gated(*wide64, offsets, "silu", dtype), "gated")
            er.close(hb.expert_product(x, gate, first), *er.product(*wide64[:2], offsets, dtype), "product")
            assert torch.equal(hb.expert_gated(x, gate, up, first), hb.expert_gated(*plain, first))
            assert torch.equal(hb.expert_product(x, gate, first), hb.expert_product(*plain[:2], first))
            dy = dy_wide[:, 3:]
            got = [*hb.expert_gated_grad(dy, x, gate, up, first), *hb.expert_product_grad(dy, x, gate, first)]
            dy = dy.contiguous()
            want = [*hb.expert_gated_grad(dy, *plain, first), *hb.expert_product_grad(dy, *plain[:2], first)]
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    x, gate, up = wide[:, :width].contiguous(), both[0, :hidden], both[0, hidden:]
    one = torch.tensor([0, rows], dtype=torch.int32, device=cuda)
    assert torch.equal(hb.expert_gated(x, gate, up), hb.expert_gated(x, gate[None], up[None], one))
    got = hb.expert_gated_grad(dy, x, gate, up)
    assert got[1].shape == gate.shape
    assert all(torch.equal(a.view(b.shape), b) for a, b in zip(got, hb.expert_gated_grad(dy, x, gate[None], up[None], one)))


def test_offsets_of_any_content(hb, cuda):
    """Offsets are read as their running maximum inside the rows: what they hold never leads outside."""
    gen = torch.Generator(device=cuda).manual_seed(4)
    for rows in (12, 200, 1500):
        for dtype in (torch.float32, torch.bfloat16):
            x, dy = (torch.randn((rows, 64), generator=gen, device=cuda).to(dtype) for _ in range(2))
            w = torch.randn((3, 64, 64), generator=gen, device=cuda).to(dtype)
            for bad, good in (([5, rows // 2, 3, rows + 7], [0, rows // 2, rows // 2, rows]), ([0, -4, 6, 2], [0, 0, 6, 6]),
                              ([-2 ** 31, 2 ** 31 - 1, 0, -1], [0, rows, rows, rows])):
                b, g = (torch.tensor(v, dtype=torch.int32, device=cuda) for v in (bad, good))
                assert torch.equal(hb.expert_product(x, w, b), hb.expert_product(x, w, g))
                assert torch.equal(hb.expert_gated(x, w, w, b), hb.expert_gated(x, w, w, g))
                for p, q in zip(hb.expert_gated_grad(dy, x, w, w, b), hb.expert_gated_grad(dy, x, w, w, g)):
                    assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("rows", [0, 5, 200])
def test_autograd(hb, cuda, dtype, rows):
    """backward() gives the gradient calls' values, each input alone too, and from no rows zeros."""
    gen = torch.Generator(device=cuda).manual_seed(rows)
    x, dy = (torch.randn((rows, 40), generator=gen, device=cuda).to(dtype) for _ in range(2))
    gate, up = (torch.randn((3, 40, 40), generator=gen, device=cuda).to(dtype) for _ in range(2))
    first = torch.tensor([0, rows // 4, rows // 2, rows], dtype=torch.int32, device=cuda)
    want = hb.expert_gated_grad(dy, x, gate, up, first)
    for on in ((True, True, True), (True, False, False), (False, True, False), (False, False, True)):
        leaves = [v.clone().requires_grad_(o) for v, o in zip((x, gate, up), on)]
        hb.expert_gated(*leaves, first).backward(dy)
        for leaf, o, w in zip(leaves, on, want):
            assert (leaf.grad is not None) == o
            if o:
                assert torch.equal(leaf.grad, w)
    want = hb.expert_product_grad(dy, x, gate, first)
    for on in ((True, True), (True, False), (False, True)):
        leaves = [v.clone().requires_grad_(o) for v, o in zip((x, gate), on)]
        hb.expert_product(*leaves, first).backward(dy)
        for leaf, o, w in zip(leaves, on, want):
            assert (leaf.grad is not None) == o and (not o or torch.equal(leaf.grad, w))
    if rows == 0:
        assert not want[1].any() and want[0].shape == (0, 40)


def test_gradients_by_differences(hb, cuda):
    """Central differences of the fp32 layer: off by h^2 / 6 of the third derivative and 2^-24 of the loss by h."""
    gen = torch.Generator(device=cuda).manual_seed(8)
    x, dy = (torch.randn((50, 20), generator=gen, device=cuda) for _ in range(2))
    gate, up = (torch.randn((2, 20, 20), generator=gen, device=cuda) / 20 ** 0.5 for _ in range(2))
    first = torch.tensor([0, 20, 50], dtype=torch.int32, device=cuda)

    def loss(values, act):
        return float((hb.expert_gated(*values, first, activation=act).double() * dy.double()).sum())

    for act in ("silu", "gelu"):
        grads = hb.expert_gated_grad(dy, x, gate, up, first, activation=act)
        for i, g in enumerate(grads):
            way = torch.randn(g.shape, generator=gen, device=cuda)
            along = float((g.double() * way.double()).sum())
            h = 2.0 ** -9
            values = [[v + s * h * way if j == i else v for j, v in enumerate((x, gate, up))] for s in (1, -1)]
            slope = (loss(values[0], act) - loss(values[1], act)) / (2 * h)
            scale = float((hb.expert_gated(x, gate, up, first, activation=act).abs() * dy.abs()).sum())
            # rounding: 1000 outputs of 20-term sums, each 2^-19 of its magnitude; curvature: h^2 of a few times the slope's size
            assert abs(slope - along) <= 2.0 ** -19 * scale / h + 8 * h * h * (float(g.abs().sum()) + scale)


def test_graph_stream_and_two_at_once(hb, cuda):
    gen = torch.Generator(device=cuda).manual_seed(5)
    jobs = []
    for rows in (6, 300, 2000):
        x, dy = (torch.randn((rows, 128), generator=gen, device=cuda).to(torch.bfloat16) for _ in range(2))
        w = [torch.randn((4, 128, 128), generator=gen, device=cuda).to(torch.bfloat16) for _ in range(2)]
        first = torch.tensor([0, rows // 5, rows // 2, rows // 2, rows], dtype=torch.int32, device=cuda)
        jobs.append((x, dy, *w, first))

    def work(x, dy, gate, up, first):
        return [hb.expert_gated(x, gate, up, first), *hb.expert_gated_grad(dy, x, gate, up, first), hb.expert_product(x, gate, first),
                *hb.expert_product_grad(dy, x, gate, first)]

    want = [work(*job) for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(5):
        got = []
        for stream, job in zip(streams, jobs):
            with torch.cuda.stream(stream):
                got.append(work(*job))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    for job in jobs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work(*job)
        for _ in range(3):
            job[0].normal_(generator=gen)
            job[4][1:4] = torch.sort(torch.randint(0, job[0].shape[0] + 1, (3,), generator=gen, device=cuda)).values
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, work(*job)))


def test_refusals(hb, cuda):
    x, w = torch.ones((4, 8), device=cuda), torch.ones((2, 6, 8), device=cuda)
    first = torch.tensor([0, 2, 4], dtype=torch.int32, device=cuda)
    for call in (lambda: hb.expert_product(x, w), lambda: hb.expert_product(x, w, first.long()), lambda: hb.expert_product(x, w, first[:2]),
                 lambda: hb.expert_product(x.half(), w, first), lambda: hb.expert_product(x.double(), w.double(), first),
                 lambda: hb.expert_product(x[:, :5], w, first), lambda: hb.expert_product(x[0], w, first),
                 lambda: hb.expert_product(x, w[0, 0], first), lambda: hb.expert_product(x.cpu(), w, first),
                 lambda: hb.expert_product(x, w, first.cpu()), lambda: hb.expert_gated(x, w, w[:, :5], first),
                 lambda: hb.expert_gated(x, w, w.half(), first), lambda: hb.expert_gated(x, w, w, first, activation="relu"),
                 lambda: hb.expert_gated(x, w, w, first, activation=None),
                 lambda: hb.expert_product(x, torch.ones((2100, 6, 8), device=cuda), torch.zeros(2101, dtype=torch.int32, device=cuda)),
                 lambda: hb.expert_product_grad(torch.ones((4, 5), device=cuda), x, w, first),
                 lambda: hb.expert_product_grad(torch.ones((3, 6), device=cuda), x, w, first),
                 lambda: hb.expert_gated_grad(torch.ones((4, 6), device=cuda).half(), x, w, w, first),
                 lambda: hb.expert_product(x[:, :0], w[:, :, :0], first)):
        with pytest.raises(ValueError):
            call()
