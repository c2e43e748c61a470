"""Table lookups and their gradient against plain 64-bit forms (bounds: tests/rows_reference.py)."""
import numpy as np
import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("n,rows,width", [(1, 1, 1), (5, 100, 2048), (33, 7, 9), (300, 50, 129), (1000, 300, 1000),
                                          (2000, 4000, 8), (1500, 100, 520), (1, 3, 9001)])
def test_lookup_matches_64_bits(hb, cuda, dtype, n, rows, width):
    rng = np.random.default_rng(n + width)
    table = torch.as_tensor(rng.normal(size=(rows, width)), device=cuda).to(dtype)
    ids = rng.integers(-2, rows + 2, n).astype(np.int32 if n % 2 else np.int64)
    scale = float(np.sqrt(width))
    live = (ids >= 0) & (ids < rows)
    want = np.zeros((n, width))
    want[live] = ref.f64(table)[ids[live]] * scale
    u = ref.U[dtype]
    got = hb.embedding_lookup(table, torch.as_tensor(ids, device=cuda), scale=scale)
    # the scale and the product are rounded to fp32 each
    ref.assert_within(got, want, ((2 * ref.E32) * (1 + u) + u) * np.abs(want) + ref.FLOOR[dtype])
    plain = hb.embedding_lookup(table, torch.as_tensor(ids, device=cuda))
    want[live] = ref.f64(table)[ids[live]]
    assert np.array_equal(ref.f64(plain), want)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("n,rows,width", [(20_000, 500, 2048), (30_000, 3000, 256), (100_000, 700, 33),
                                          (200_000, 100, 8)])
def test_lookup_of_many_rows(hb, cuda, dtype, n, rows, width):
    """Scaled by 2, which is exact: equal to indexing, bit for bit."""
    gen = torch.Generator(device=cuda).manual_seed(n)
    table = torch.randn((rows, width), generator=gen, device=cuda).to(dtype)
    ids = torch.randint(-1, rows, (n,), generator=gen, device=cuda)
    want = torch.where((ids >= 0).unsqueeze(1), 2 * table[ids.clamp(min=0)], torch.zeros((), dtype=dtype, device=cuda))
    assert torch.equal(hb.embedding_lookup(table, ids, scale=2), want)


def _grad_reference(dy, ids, rows, scale):
    want, mag, count = (np.zeros((rows, dy.shape[1])) for _ in range(3))
    live = (ids >= 0) & (ids < rows)
    np.add.at(want, ids[live], dy[live] * scale)
    np.add.at(mag, ids[live], np.abs(dy[live] * scale))
    np.add.at(count, ids[live], 1)
    return want, mag, count


IDS = {
    "spread": lambda rng, n, rows: rng.integers(0, rows, n),
    "one row": lambda rng, n, rows: np.full(n, rows - 1),
    "frequent": lambda rng, n, rows: np.minimum(rows - 1, (rows ** rng.random(n)).astype(np.int64) - 1),
    "outside": lambda rng, n, rows: rng.integers(-rows, 2 * rows, n),
    "none": lambda rng, n, rows: np.full(n, -1),
    "distinct": lambda rng, n, rows: rng.permutation(max(n, rows))[:n],
}


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("kind", IDS)
@pytest.mark.parametrize("n,rows,width", [(1, 1, 1), (1, 5000, 7), (65, 3, 16), (1000, 503, 129), (700, 40, 2048),
                                          (5000, 100, 264), (6000, 3000, 33), (300, 9, 4104)])
def test_grad_matches_64_bits(hb, cuda, dtype, kind, n, rows, width):
    rng = np.random.default_rng(n + rows + width)
    ids = np.asarray(IDS[kind](rng, n, rows), dtype=np.int64)
    dy = torch.as_tensor(rng.normal(size=(n, width)), device=cuda).to(dtype)
    scale = 1.7
    want, mag, count = _grad_reference(ref.f64(dy), ids, rows, scale)
    for out_type in {dtype, torch.float32}:
        u = ref.U[out_type]
        bound = (count + 2) * ref.E32 * mag * (1 + u) + u * np.abs(want) + ref.FLOOR[out_type]
        t = torch.as_tensor(ids, device=cuda)
        got = hb.embedding_grad(dy, t, rows, scale=scale, dtype=out_type)
        ref.assert_within(got, want, bound, kind)
        assert torch.equal(got, hb.embedding_grad(dy, t.to(torch.int32), rows, scale=scale, dtype=out_type))
        # into a gradient that is there already: other rows stay as they are, bit for bit
        base = torch.as_tensor(rng.normal(size=(rows, width)), device=cuda).to(out_type)
        total = base.clone()
        assert hb.embedding_grad(dy, t, rows, scale=scale, out=total, accumulate=True) is total
        both = ref.f64(base) + want
        ref.assert_within(total, both, (count + 3) * ref.E32 * (mag + np.abs(ref.f64(base))) * (1 + u) + u * np.abs(both)
                          + ref.FLOOR[out_type], kind)
        untouched = torch.as_tensor(count[:, 0] == 0, device=cuda)
        assert torch.equal(total[untouched], base[untouched])


@pytest.mark.parametrize("n,rows,width", [(150_000, 5000, 256), (600_000, 70_000, 8), (40_000, 200, 16), (300_000, 3, 4)])
def test_grad_of_long_runs_and_large_batches(hb, cuda, n, rows, width):
    """Enough tokens for long chunks and several sort tiles; one row takes a third of them."""
    gen = torch.Generator(device=cuda).manual_seed(4)
    ids = torch.randint(0, rows, (n,), generator=gen, device=cuda)
    ids[torch.rand(n, generator=gen, device=cuda) < 1 / 3] = 2
    dy = torch.randn((n, width), generator=gen, device=cuda).to(torch.bfloat16)
    got = hb.embedding_grad(dy, ids, rows, dtype=torch.float32)
    want = torch.zeros((rows, width), dtype=torch.float64, device=cuda).index_add_(0, ids, dy.double())
    mag = torch.zeros((rows, width), dtype=torch.float64, device=cuda).index_add_(0, ids, dy.double().abs())
    count = torch.bincount(ids, minlength=rows).double().unsqueeze(1)
    assert bool(((got.double() - want).abs() <= (count + 2) * ref.E32 * mag).all())
    assert torch.equal(got, hb.embedding_grad(dy, ids, rows, dtype=torch.float32))  # nothing depends on the launch


def test_strides_addresses_and_shapes(hb, cuda):
    gen = torch.Generator(device=cuda).manual_seed(2)
    wide = torch.randn((90, 300), generator=gen, device=cuda)
    ids = torch.randint(0, 90, (4, 15), generator=gen, device=cuda)
    for table in (wide[:, :256], wide[:, 1:258], wide[:, 2:12], wide.t()[:90, :90]):
        y = hb.embedding_lookup(table, ids, scale=2.0)
        assert y.shape == (4, 15, table.shape[1]) and torch.equal(y, table[ids] * 2.0)
        assert torch.equal(hb.embedding_lookup(table, ids.t(), scale=2.0), (table[ids] * 2.0).transpose(0, 1))
        dy = table[:60].view(4, 15, -1) if table.stride(1) == 1 else table[:60].reshape(4, 15, -1)
        assert torch.equal(hb.embedding_grad(dy, ids, 90), hb.embedding_grad(dy.contiguous().clone(), ids, 90))
    one = torch.ones((), device=cuda).expand(60, 8)  # the gradient of a sum
    want = torch.bincount(ids.view(-1), minlength=90).float().unsqueeze(1).expand(90, 8)
    assert torch.equal(hb.embedding_grad(one, ids.view(-1), 90), want)
    off = torch.zeros(90 * 8 + 1, device=cuda)[1:].view(90, 8)  # an output off the 16-byte grid
    hb.embedding_grad(one, ids.view(-1), 90, out=off)
    assert torch.equal(off, want)
    none = torch.empty((0,), dtype=torch.int64, device=cuda)
    assert hb.embedding_lookup(wide, none).shape == (0, 300)
    assert not hb.embedding_grad(torch.empty((0, 8), device=cuda), none, 5).any()
    kept = torch.ones((5, 8), device=cuda)
    hb.embedding_grad(torch.empty((0, 8), device=cuda), none, 5, out=kept, accumulate=True)
    assert bool((kept == 1).all())


def test_nonfinite_rows_stay_their_own(hb, cuda):
    """An infinity or NaN in one token's row reaches its own table row alone."""
    dy = torch.ones((100, 16), device=cuda)
    ids = torch.arange(100, device=cuda) // 10
    dy[35], dy[50, 3], dy[99] = float("inf"), float("nan"), float("nan")
    ids[99] = -1
    got = hb.embedding_grad(dy, ids, 12)
    assert bool(torch.isinf(got[3]).all()) and bool(torch.isnan(got[5, 3])) and bool((got[9] == 9).all())
    good = [0, 1, 2, 4, 6, 7, 8]
    assert bool((got[good] == 10).all()) and not got[10:].any()


def test_autograd_and_differences(hb, cuda):
    """The gradient of sum(r * lookup) through autograd, against the change of the loss along a direction; the
    lookup is linear, so the difference is exact up to the fp32 rounding of its values."""
    rng = np.random.default_rng(8)
    rows, width, n = 20, 12, 70
    ids = rng.integers(-1, rows, n)
    table = torch.as_tensor(rng.normal(size=(rows, width)), dtype=torch.float32, device=cuda).requires_grad_()
    r = torch.as_tensor(rng.normal(size=(n, width)), dtype=torch.float32, device=cuda)
    t = torch.as_tensor(ids, device=cuda)
    (hb.embedding_lookup(table, t, scale=0.5) * r).sum().backward()
    for _ in range(4):
        v = torch.as_tensor(rng.normal(size=(rows, width)), dtype=torch.float32, device=cuda)
        with torch.no_grad():
            change = sum(s * float((hb.embedding_lookup(table + s * v, t, scale=0.5).double() * r.double()).sum())
                         for s in (1, -1)) / 2
        along = float((table.grad.double() * v.double()).sum())
        scale = float(np.abs(ref.f64(table)).max() + 4) * float(r.abs().sum())
        assert abs(along - change) <= 2.0 ** -22 * scale


def test_written_gradients_count_as_changed(hb, cuda):
    out = torch.zeros((5, 4), device=cuda)
    before = out._version
    hb.embedding_grad(torch.ones((3, 4), device=cuda), torch.tensor([0, 1, 1], device=cuda), 5, out=out)
    assert out._version > before


def test_refusals(hb, cuda):
    table, ids, dy = (torch.zeros((6, 4), device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda),
                      torch.zeros((3, 4), device=cuda))
    for call in (lambda: hb.embedding_lookup(table.double(), ids), lambda: hb.embedding_lookup(table, ids.float()),
                 lambda: hb.embedding_lookup(table[0], ids), lambda: hb.embedding_lookup(table.cpu(), ids),
                 lambda: hb.embedding_lookup(table, ids.cpu()), lambda: hb.embedding_grad(dy, ids[:2], 6),
                 lambda: hb.embedding_grad(dy, ids, 0), lambda: hb.embedding_grad(dy, ids, 6, dtype=torch.float16),
                 lambda: hb.embedding_grad(dy, ids, 6, accumulate=True),
                 lambda: hb.embedding_grad(dy, ids, 6, out=table[:5]),
                 lambda: hb.embedding_grad(dy, ids, 6, out=table.t().contiguous().t()),
                 lambda: hb.embedding_grad(dy.half(), ids, 6, out=table.to(torch.bfloat16))):
        with pytest.raises(ValueError):
            call()
