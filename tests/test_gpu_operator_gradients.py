"""Gradients where other tests do not reach: long chunks of short vectors, groups smaller than a warp, and autograd in
every type (bounds: tests/rows_reference.py)."""
import numpy as np
import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,rows,width,dtype", [
    (46_656, 1120, 187, torch.float32), (92_503, 105_992, 369, torch.float32), (150_000, 50, 3, torch.float32),   # 4-byte vectors
    (40_000, 30_000, 1002, torch.float16), (40_000, 300, 514, torch.bfloat16), (120_000, 40, 6, torch.bfloat16),
    (40_000, 30_000, 1001, torch.bfloat16), (40_000, 200, 9, torch.float16), (300_000, 7, 1, torch.bfloat16),     # 2-byte vectors
    (60_000, 500, 308, torch.float16), (60_000, 90, 12, torch.bfloat16), (50_000, 400, 50, torch.float32)])       # 8-byte vectors
def test_long_chunks_of_short_vectors(hb, cuda, n, rows, width, dtype):
    """Off the 16-byte grid with enough tokens for chunks of more than 16 places; one row takes a third of them."""
    gen = torch.Generator(device=cuda).manual_seed(n + width)
    ids = torch.randint(-1, rows, (n,), generator=gen, device=cuda)
    ids[torch.rand(n, generator=gen, device=cuda) < 1 / 3] = rows // 2
    dy = torch.randn((n, width), generator=gen, device=cuda).to(dtype)
    scale, live = 1.25, ids >= 0
    d64 = dy[live].double() * scale
    want = torch.zeros((rows, width), dtype=torch.float64, device=cuda).index_add_(0, ids[live], d64)
    mag = torch.zeros_like(want).index_add_(0, ids[live], d64.abs())
    count = torch.bincount(ids[live], minlength=rows).double().unsqueeze(1)
    del d64
    for out_type in {dtype, torch.float32}:
        u = ref.U[out_type]
        got = hb.embedding_grad(dy, ids, rows, scale=scale, dtype=out_type)
        bound = (count + 2) * ref.E32 * mag * (1 + u) + u * want.abs() + ref.FLOOR[out_type]
        assert bool(((got.double() - want).abs() <= bound).all())
        assert torch.equal(got, hb.embedding_grad(dy, ids, rows, scale=scale, dtype=out_type))
        base = torch.randn((rows, width), generator=gen, device=cuda).to(out_type)
        total = base.clone()
        hb.embedding_grad(dy, ids, rows, scale=scale, out=total, accumulate=True)
        both = base.double() + want
        bound = (count + 3) * ref.E32 * (mag + base.double().abs()) * (1 + u) + u * both.abs() + ref.FLOOR[out_type]
        assert bool(((total.double() - both).abs() <= bound).all())
        untouched = count[:, 0] == 0
        assert torch.equal(total[untouched], base[untouched])


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("tokens,slots,experts,width", [(37, 3, 5, 40), (700, 2, 9, 129), (5000, 1, 16, 64)])
def test_autograd_in_every_type(hb, cuda, dtype, tokens, slots, experts, width):
    """Gradients of lookup, dispatch and combine through backward(), against their formulas in 64 bits."""
    rng = np.random.default_rng(tokens)
    index = rng.integers(-1, experts, (tokens, slots))
    plan = hb.route_plan(torch.as_tensor(index, device=cuda), experts)
    order, position, offsets = ref.plan(index, experts)
    kept, live = int(offsets[-1]), order[:int(offsets[-1])]
    u, floor = ref.U[dtype], ref.FLOOR[dtype]

    def data(*shape):
        return torch.as_tensor(rng.normal(size=shape), device=cuda).to(dtype)

    # lookup
    table, ids, dy = data(30, width).requires_grad_(), rng.integers(-1, 30, tokens), data(tokens, width)
    hb.embedding_lookup(table, torch.as_tensor(ids, device=cuda), scale=1.5).backward(dy)
    assert table.grad.dtype == dtype
    want, mag, count = np.zeros((30, width)), np.zeros((30, width)), np.zeros((30, 1))
    np.add.at(want, ids[ids >= 0], ref.f64(dy)[ids >= 0] * 1.5)
    np.add.at(mag, ids[ids >= 0], np.abs(ref.f64(dy)[ids >= 0] * 1.5))
    np.add.at(count, ids[ids >= 0], 1)
    ref.assert_within(table.grad, want, (count + 2) * ref.E32 * mag * (1 + u) + u * np.abs(want) + floor, "table")
    # dispatch
    x, dxs = data(tokens, width).requires_grad_(), data(tokens * slots, width)
    hb.route_dispatch(x, plan).backward(dxs)
    want, mag = ref.combine(ref.f64(dxs), position, kept, None)
    assert x.grad.dtype == dtype
    ref.assert_within(x.grad, want, slots * ref.E32 * mag * (1 + u) + u * np.abs(want) + floor, "x")
    # combine, with weights of its own type and of fp32, and each of the two gradients alone
    for weight_type in {dtype, torch.float32}:
        z = data(tokens * slots, width)
        w = torch.as_tensor(rng.random((tokens, slots)), device=cuda).to(weight_type)
        dz64, dw64, dw_mag = np.zeros((tokens * slots, width)), np.zeros(tokens * slots), np.zeros(tokens * slots)
        dz64[:kept] = ref.f64(dy)[live // slots] * ref.f64(w).reshape(-1)[live][:, None]
        pairs = ref.f64(dy)[live // slots] * ref.f64(z)[:kept]
        dw64[live], dw_mag[live] = pairs.sum(1), np.abs(pairs).sum(1)
        uw = ref.U[weight_type]
        for with_z, with_w in ((True, True), (True, False), (False, True)):
            z_, w_ = z.clone().requires_grad_(with_z), w.clone().requires_grad_(with_w)
            hb.route_combine(z_, plan, w_).backward(dy)
            assert (z_.grad is not None) == with_z and (w_.grad is not None) == with_w
            if with_z:
                ref.assert_within(z_.grad, dz64, (ref.E32 * (1 + u) + u) * np.abs(dz64) + floor, "z")
            if with_w:
                assert w_.grad.dtype == weight_type
                ref.assert_within(w_.grad.view(-1), dw64, width * ref.E32 * dw_mag * (1 + uw) + uw * np.abs(dw64)
                                  + ref.FLOOR[weight_type], "weights")
