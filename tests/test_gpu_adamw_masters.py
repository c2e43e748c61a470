"""Masters of fp32 parameters: a step starts from the master, whatever the parameter holds."""
import pytest
import torch

pytestmark = pytest.mark.gpu
RULE = dict(lr=2e-3, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.05)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("size", [1, 255, 5000, 40_001])
def test_master_of_an_fp32_parameter(hb, cuda, size, bits):
    gen = torch.Generator(device=cuda).manual_seed(size + bits)

    def normal():
        return torch.randn(size, generator=gen, device=cuda)

    held, other, grads = normal(), normal(), [normal(), normal()]
    alone = [held.clone(), other.clone()]
    params, master = [normal(), other.clone()], held.clone()  # the second parameter has no master
    state = hb.adamw_state(params, bits=bits)._replace(master=[master, None])
    plain = hb.adamw_state(alone, bits=bits)
    for _ in range(2):
        hb.adamw_step(params, grads, state, **RULE)
        hb.adamw_step(alone, grads, plain, **RULE)
        assert torch.equal(master, alone[0]) and torch.equal(params[0], master) and torch.equal(params[1], alone[1])
        params[0].zero_()
