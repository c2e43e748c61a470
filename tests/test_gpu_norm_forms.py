"""The row norm where its forms differ: the sum without a residual, gradients of rows of very large and very small values,
every width that has a kernel of its own, views in 8 bits."""
import pytest
import torch

import rows_reference as ref
import test_gpu_norm as base
from expert_reference import close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("width", [7, 2048, 16384, 16385, 16400])
def test_sum_without_a_residual(hb, cuda, width, dtype):
    """The C entry's `total` is the rows themselves then, in the held form and in that of wider rows, with y and with codes."""
    lib, types = hb.load_library(), {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    x, _, w, _, _ = base._data(cuda, 5, width, dtype, dtype, False)
    stream = torch.cuda.current_stream().cuda_stream
    for eight in (False, True):
        total, y = torch.full_like(x, float("nan")), torch.empty_like(x)
        codes = torch.empty((5, width), dtype=torch.uint8, device=cuda)
        scales = torch.empty((5, -(-width // 32)), dtype=torch.uint8, device=cuda)
        assert lib.hb_rms_norm(types[dtype], x.data_ptr(), width, None, 0, 5, width, w.data_ptr(), types[dtype], base.EPS,
                               None if eight else y.data_ptr(), codes.data_ptr() if eight else None, scales.data_ptr() if eight else None,
                               total.data_ptr(), stream) == hb._lib.HB_OK
        assert torch.equal(total, x)
        if eight:
            want = hb.rms_norm_8bit(x, w, eps=base.EPS)[0]
            assert torch.equal(codes, want.values.view(torch.uint8)) and torch.equal(scales, want.scales.view(torch.uint8))
        else:
            assert torch.equal(y, hb.rms_norm(x, w, eps=base.EPS))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [7, 64, 2048, 16400])
@pytest.mark.parametrize("size,eps", [(1e15, 1e-6), (1e17, 1e-6), (1e-14, 0.0), (1e-17, 0.0)])
def test_gradients_of_large_and_small_rows(hb, cuda, size, eps, width, dtype):
    """The row's length enters dx to the third power, which fp32 does not hold where it holds the squares' sum.  Bounds as in
    test_gradients: the same sums, and fewer than 12 roundings beside them.  dy lies along x, so that the term counts."""
    x, _, w, noise, _ = base._data(cuda, 3, width, dtype, torch.float32, scale=size)
    dy = (x.double() / size + 0.25 * noise.double()).to(dtype)
    x64, w64, g64 = x.double(), w.double(), dy.double()
    inverse = (x64.square().mean(1, keepdim=True) + eps).rsqrt()
    pull = (w64 * g64 * x64).mean(1, keepdim=True)
    want = inverse * w64 * g64 - x64 * inverse ** 3 * pull
    each, u = (width + 12) * ref.E32, ref.U[dtype]
    mag = inverse * (w64 * g64).abs() + x64.abs() * inverse ** 3 * (w64 * g64 * x64).abs().mean(1, keepdim=True)
    bound = 3 * each * mag + 2 * ref.E32 * want.abs()
    dx, dw = hb.rms_norm_grad(dy, x, w, eps=eps)
    close(dx, want, bound * (1 + u) + u * want.abs() + ref.FLOOR[dtype], "dx")
    terms = g64 * x64 * inverse
    close(dw, terms.sum(0), (3 + width / 2 + 12) * ref.E32 * terms.abs().sum(0) + ref.E32 * terms.sum(0).abs(), "dw")


# widths of each kernel's own: 2049 to 4096, 4097 to 8192 and 8193 to 16384 columns on and off the 16-byte grid, rows enough for
# several of a block, in order (forward) and strided (gradients)
FORMS = [(5, 4096), (5, 8192), (7, 1090), (7, 1091), (5, 3333), (5, 6002), (4, 12001), (40003, 64), (3001, 2048)]


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("rows,width", FORMS)
def test_forms(hb, cuda, rows, width, dtype):
    base.test_forward(hb, cuda, rows, width, dtype)
    base.test_gradients(hb, cuda, rows, width, dtype)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("width", [128, 101, 1090, 4500])
def test_strides_in_8_bits(hb, cuda, width, dtype):
    """Rows apart, off the grid, in another order, the same one again: the values that the codes stand for, within the
    bounds of test_forward, and scales from both sides."""
    x, r, w, _, _ = base._data(cuda, 40, width + 4, dtype, dtype)
    for view in (lambda v: v[:, :width], lambda v: v[:, 2:width + 2], lambda v: v[:, 1:width + 1], lambda v: v.t().contiguous().t()[:, :width],
                 lambda v: v[:1, :width].expand(40, width), lambda v: v[::2, :width]):
        a, b, k = view(x), view(r), w[:width]
        t = a.double() + b.double()
        want = base._norm(t, k.double())
        rows8, total = hb.rms_norm_8bit(a, k, b, eps=base.EPS)
        close(total, t, ref.E32 * t.abs() + ref.U[dtype] * t.abs() * (1 + ref.E32) + ref.FLOOR[dtype], "sum")
        most = torch.nn.functional.pad(want.abs(), (0, -width % 32)).view(len(want), -1, 32).amax(-1)
        off = 1 + (width / 2 + 8) * ref.E32
        floor = (2 * most * off / 448 * 2.0 ** -10).repeat_interleave(32, 1)[:, :width]
        close(hb.rows_of_8bit(rows8), want, 2.0 ** -4 * want.abs() * off + floor + (width / 2 + 8) * ref.E32 * want.abs(), "8 bits")
        scale = rows8.scales.float()
        assert bool((scale >= most / 448 * (2 - off)).all()) and bool((scale < 2 * most / 448 * off).all())
    # codes and scales that lie apart are read as their dense copies
    wide = hb.rms_norm_8bit(x, w, r, eps=base.EPS)[0]
    apart = (wide.values.view(torch.uint8).repeat(1, 2)[:, :width + 4].view(torch.float8_e4m3fn),
             wide.scales.view(torch.uint8).repeat(1, 2)[:, :wide.scales.shape[1]].view(torch.float8_e8m0fnu))
    assert not apart[0].is_contiguous() and torch.equal(hb.rows_of_8bit(apart), hb.rows_of_8bit(wide))
