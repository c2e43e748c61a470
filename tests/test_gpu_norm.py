"""Root-mean-square norm, its 8-bit output and its gradients against 64-bit forms.

Bounds: t = x + residual is off by 2^-24 of itself, its sum of squares by (d + 2) 2^-24, the root, quotient and
products by at most 4 2^-24 more, so y by (d / 2 + 8) 2^-24 of itself, and U of it where it is rounded.
"""
import pytest
import torch

import rows_reference as ref
from expert_reference import close

pytestmark = pytest.mark.gpu
EPS = 1e-5
SIZES = [(1, 1), (3, 7), (5, 2048), (130, 64), (70, 513), (33, 1000), (9, 1536), (6, 4097), (4, 16384), (3, 16400), (2, 40001), (700, 32)]


def _data(cuda, rows, width, dtype, weight_type, residual=True, scale=1.0):
    gen = torch.Generator(device=cuda).manual_seed(rows * 100 + width)

    def normal(*size):
        return torch.randn(size, generator=gen, device=cuda)

    x, r = (normal(rows, width) * scale).to(dtype), (normal(rows, width) * scale).to(dtype) if residual else None
    return x, r, (1 + 0.3 * normal(width)).to(weight_type), normal(rows, width).to(dtype), normal(rows, width).to(dtype)


def _norm(t, w, eps=EPS):
    return t / (t.square().mean(-1, keepdim=True) + eps).sqrt() * w


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("rows,width", SIZES)
def test_forward(hb, cuda, rows, width, dtype):
    for weight_type, with_residual in ((dtype, True), (torch.float32, False), (torch.float16, True)):
        x, r, w, _, _ = _data(cuda, rows, width, dtype, weight_type, with_residual)
        t = x.double() + (r.double() if with_residual else 0)
        got = hb.rms_norm(x, w, r, eps=EPS)
        if with_residual:
            got, total = got
            assert total.dtype == dtype
            close(total, t, ref.E32 * t.abs() + ref.U[dtype] * t.abs() * (1 + ref.E32) + ref.FLOOR[dtype], "sum")
        want = _norm(t, w.double())
        assert got.dtype == dtype
        close(got, want, ((width / 2 + 8) * ref.E32 * (1 + ref.U[dtype]) + ref.U[dtype]) * want.abs() + ref.FLOOR[dtype], "y")
        # in 8 bits: half a step of e4m3, 2^-4 of the value or 2^-10 of the scale, which is less than 2 / 448 of the group's largest
        rows8, total8 = hb.rms_norm_8bit(x, w, r, eps=EPS)
        assert rows8.values.dtype == torch.float8_e4m3fn and rows8.scales.shape == (rows, -(-width // 32))
        assert total8 is None if not with_residual else torch.equal(total8, total)
        back = hb.rows_of_8bit(rows8)
        groups = torch.nn.functional.pad(want.abs(), (0, -width % 32)).view(rows, -1, 32)
        most = groups.amax(-1)
        off = 1 + (width / 2 + 8) * ref.E32
        floor = (2 * most * off / 448 * 2.0 ** -10).repeat_interleave(32, 1)[:, :width]
        close(back, want, 2.0 ** -4 * want.abs() * off + floor + (width / 2 + 8) * ref.E32 * want.abs(), "8 bits")
        scale = rows8.scales.float()
        least = torch.where(most > 0, most / 448, torch.zeros_like(most))
        assert bool((scale >= least * (2 - off)).all()) and bool(((scale < 2 * least * off) | (most == 0)).all())
        for out_type in ref.DTYPES:
            assert torch.equal(hb.rows_of_8bit(rows8, dtype=out_type), back.to(out_type))


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("rows,width", SIZES)
def test_gradients(hb, cuda, rows, width, dtype):
    """dx carries two sums of width terms; their errors are relative to the sums of magnitudes."""
    for weight_type, with_dsum in ((dtype, True), (torch.float32, False)):
        x, _, w, dy, dsum = _data(cuda, rows, width, dtype, weight_type)
        x64, w64, g64 = x.double(), w.double(), dy.double()
        inverse = (x64.square().mean(1, keepdim=True) + EPS).rsqrt()
        pull = (w64 * g64 * x64).mean(1, keepdim=True)
        want = inverse * w64 * g64 - x64 * inverse ** 3 * pull + (dsum.double() if with_dsum else 0)
        each = (width + 12) * ref.E32
        mag = inverse * (w64 * g64).abs() + x64.abs() * inverse ** 3 * (w64 * g64 * x64).abs().mean(1, keepdim=True)
        bound = 3 * each * mag + 2 * ref.E32 * want.abs()
        dx, dw = hb.rms_norm_grad(dy, x, w, dsum=dsum if with_dsum else None, eps=EPS)
        assert dx.dtype == dtype and dw.dtype == weight_type
        u = ref.U[dtype]
        if with_dsum:
            bound = bound + ref.E32 * (want.abs() + dsum.double().abs())
        close(dx, want, bound * (1 + u) + u * want.abs() + ref.FLOOR[dtype], "dx")
        terms = g64 * x64 * inverse
        want_w, u = terms.sum(0), ref.U[weight_type]
        close(dw, want_w, (rows + width / 2 + 12) * ref.E32 * terms.abs().sum(0) * (1 + u) + u * want_w.abs() + ref.FLOOR[weight_type], "dw")
        for needs in ((True, False), (False, True)):
            part = hb.rms_norm_grad(dy, x, w, dsum=dsum if with_dsum else None, eps=EPS, needs=needs)
            for need, p, full in zip(needs, part, (dx, dw)):
                assert torch.equal(p, full) if need else p is None


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_autograd_and_shapes(hb, cuda, dtype):
    x, r, w, dy, dsum = (v.clone() for v in _data(cuda, 24, 96, dtype, dtype))
    shape = (2, 3, 4, 96)
    want = hb.rms_norm_grad(dy, hb.rms_norm(x, w, r)[1], w, dsum=dsum)
    leaves = [v.clone().requires_grad_() for v in (x.view(shape), w, r.view(shape))]
    y, total = hb.rms_norm(*leaves)
    assert y.shape == total.shape == shape
    torch.autograd.backward((y, total), (dy.view(shape), dsum.view(shape)))
    assert torch.equal(leaves[0].grad.view_as(x), want[0]) and torch.equal(leaves[2].grad, leaves[0].grad)
    assert torch.equal(leaves[1].grad, want[1])
    # one output alone
    a, b = x.clone().requires_grad_(), r.clone().requires_grad_()
    hb.rms_norm(a, w, b)[1].backward(dsum)
    assert torch.equal(a.grad, dsum) and torch.equal(b.grad, dsum)
    b = r.clone().requires_grad_()
    hb.rms_norm(x, w, b)[0].backward(dy)
    assert torch.equal(b.grad, hb.rms_norm_grad(dy, hb.rms_norm(x, w, r)[1], w)[0])
    v = w.clone().requires_grad_()
    hb.rms_norm(x, v).backward(dy)
    assert torch.equal(v.grad, hb.rms_norm_grad(dy, x, w)[1])
    assert hb.rms_norm(x[0], w).shape == (96,)
    empty = hb.rms_norm(x[:0], w, r[:0])
    assert empty[0].shape == empty[1].shape == (0, 96) and hb.rms_norm_8bit(x[:0], w)[0].scales.shape == (0, 3)
    assert not hb.rms_norm_grad(dy[:0], x[:0], w)[1].any()


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_strides(hb, cuda, dtype):
    x, r, w, dy, dsum = _data(cuda, 40, 130, dtype, dtype)
    for width in (128, 101):
        for view in (lambda v: v[:, :width], lambda v: v[:, 2:width + 2], lambda v: v[:, 1:width + 1], lambda v: v.t().contiguous().t()[:, :width],
                     lambda v: v[:1, :width].expand(40, width), lambda v: v[::2, :width]):
            a, b, g, s, k = view(x), view(r), view(dy), view(dsum), w[:width]
            plain = [v.contiguous() for v in (a, b, g, s)]
            for got, want in zip((*hb.rms_norm(a, k, b), *hb.rms_norm_grad(g, a, k, dsum=s)),
                                 (*hb.rms_norm(plain[0], k, plain[1]), *hb.rms_norm_grad(plain[2], plain[0], k, dsum=plain[3]))):
                # the forms for other vectors sum in another order
                u = ref.U[dtype]
                bound = (2 * u + 1500 * ref.E32) * want.double().abs().amax(-1, keepdim=True)
                close(got, want.double(), bound, "strides")
            got, want = hb.rms_norm_8bit(a, k)[0], hb.rms_norm_8bit(plain[0], k)[0]
            assert got.values.shape == want.values.shape and bool((got.scales.float() <= 2 * want.scales.float()).all())
    odd = torch.ones(1 + 128, dtype=dtype, device=cuda)[1:]
    assert torch.equal(hb.rms_norm(x[:, :128], odd), hb.rms_norm(x[:, :128], odd.clone()))


def test_extremes(hb, cuda):
    w = torch.ones(64, device=cuda)
    for value in (0.0, 1e-30, 1e15, 1e-18):
        x = torch.full((2, 64), value, device=cuda)
        t = x.double()
        close(hb.rms_norm(x, w, eps=1e-6), _norm(t, 1.0, 1e-6), 40 * ref.E32 * _norm(t, 1.0, 1e-6) + 1e-38, value)
        rows8 = hb.rms_norm_8bit(x, w, eps=1e-6)[0]
        back, want = hb.rows_of_8bit(rows8), _norm(t, 1.0, 1e-6)
        close(back, want, 2.0 ** -3 * want + 2.0 ** -135, value)
    x = torch.ones((3, 64), device=cuda)
    x[1, 5] = float("nan")
    rows8 = hb.rms_norm_8bit(x, w)[0]
    back = hb.rows_of_8bit(rows8)
    assert bool(torch.isnan(back[1]).all()) and bool(torch.isfinite(back[[0, 2]]).all())
    assert bool(torch.isnan(hb.rms_norm(x, w)[1]).all())
    weight = w.clone()
    weight[40] = float("inf")
    back = hb.rows_of_8bit(hb.rms_norm_8bit(x[:1], weight)[0])
    assert bool(torch.isfinite(back[0, :32]).all()) and bool(torch.isnan(back[0, 32:]).all())
    # values that end a scale's range: 448 times a power of two fits, the next float does not
    for top, scale in ((448.0, 1.0), (448.0 * (1 + 2.0 ** -23), 2.0), (3.5, 2.0 ** -7), (449.0, 2.0), (256.0, 1.0), (224.0, 0.5)):
        big = torch.zeros(64, device=cuda)
        big[0] = top
        row = torch.ones((1, 64), device=cuda)
        got = hb.rms_norm_8bit(row, big, eps=0.0)[0]
        assert float(got.scales.float()[0, 0]) == scale and float(got.scales.float()[0, 1]) in (0.0, 2.0 ** -127)


def test_every_code_and_scale(hb, cuda):
    """Rows from elsewhere: each of the 256 codes with each of the 256 scales reads as the numbers that they are."""
    codes = torch.arange(256, dtype=torch.int32, device=cuda).to(torch.uint8).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.int32, device=cuda).to(torch.uint8).view(256, 1).repeat(1, 8)
    want = codes.view(torch.float8_e4m3fn).double() * torch.where(scales == 255, torch.nan, 2.0 ** (scales.double() - 127)).repeat_interleave(32, 1)
    for out_type in ref.DTYPES:
        for width in (256, 237):
            values = codes[:, :width].contiguous().view(torch.float8_e4m3fn)
            got = hb.rows_of_8bit((values, scales.view(torch.float8_e8m0fnu)), dtype=out_type)
            assert torch.equal(got.nan_to_num(7.5), want[:, :width].float().to(out_type).nan_to_num(7.5))


def test_graph_and_refusals(hb, cuda):
    x, r, w, dy, dsum = _data(cuda, 300, 256, torch.bfloat16, torch.float32)
    graph = torch.cuda.CUDAGraph()
    hb.rms_norm_grad(dy, x, w, dsum=dsum)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = [*hb.rms_norm(x, w, r), *hb.rms_norm_8bit(x, w, r)[0], *hb.rms_norm_grad(dy, x, w, dsum=dsum)]
    x.normal_()
    graph.replay()
    for a, b in zip(out, [*hb.rms_norm(x, w, r), *hb.rms_norm_8bit(x, w, r)[0], *hb.rms_norm_grad(dy, x, w, dsum=dsum)]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    rows8 = hb.rms_norm_8bit(x, w)[0]
    for call in (lambda: hb.rms_norm(x, w[:3]), lambda: hb.rms_norm(x, w[None]), lambda: hb.rms_norm(x, w, r[:2]), lambda: hb.rms_norm(x, w, r.half()),
                 lambda: hb.rms_norm(x.double(), w), lambda: hb.rms_norm(x, w, eps=-1.0), lambda: hb.rms_norm(x, w, eps=float("nan")),
                 lambda: hb.rms_norm(x[:, :0], w[:0]), lambda: hb.rms_norm(x.cpu(), w), lambda: hb.rms_norm_grad(dy[:, :8], x, w),
                 lambda: hb.rms_norm_grad(dy.float(), x, w), lambda: hb.rms_norm_grad(dy, x, w, dsum=dsum.float()),
                 lambda: hb.rows_of_8bit((rows8.values, rows8.scales[:, :1])), lambda: hb.rows_of_8bit((x, rows8.scales)),
                 lambda: hb.rows_of_8bit(rows8, dtype=torch.float64)):
        with pytest.raises(ValueError):
            call()
