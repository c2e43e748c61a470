"""The row norm where its forms differ: the sum without a residual."""
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
