"""The experts', norm and optimizer calls without a GPU: no CPU path, and what the C entries refuse before any launch
(addresses are made up and never read)."""
import ctypes
from array import array

import pytest
import torch

A = 1 << 20  # an aligned address


def test_no_cpu_path(hb, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    x, w, first = torch.zeros((4, 6)), torch.zeros((2, 5, 6)), torch.tensor([0, 2, 4], dtype=torch.int32)
    h, k = torch.zeros((4, 5)), torch.ones(6)
    state = hb.adamw_state([x])
    rows8 = hb.Rows8(torch.zeros((4, 32), dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros((4, 1), dtype=torch.uint8).view(torch.float8_e8m0fnu))
    for call in (lambda: hb.expert_product(x, w, first), lambda: hb.expert_gated(x, w, w, first), lambda: hb.expert_product_grad(h, x, w, first),
                 lambda: hb.expert_gated_grad(h, x, w, w, first), lambda: hb.rms_norm(x, k), lambda: hb.rms_norm_8bit(x, k),
                 lambda: hb.rms_norm_grad(x, x, k), lambda: hb.rows_of_8bit(rows8), lambda: hb.adamw_step([x], [x.clone()], state, lr=0.1)):
        with pytest.raises(hb.HBError, match="requires a CUDA device"):
            call()


def test_states(hb):
    p = [torch.ones((3, 100)), torch.ones(5, dtype=torch.bfloat16), torch.ones((0, 4), dtype=torch.float16)]
    s = hb.adamw_state(p, bits=8, master=True)
    assert [t.shape for t in s.exp_avg] == [v.shape for v in p] and {t.dtype for t in s.exp_avg + s.exp_avg_sq} == {torch.float8_e4m3fn}
    assert [t.numel() for t in s.exp_avg_scale] == [2, 1, 0] and int(s.step) == 0 and s.step.dtype == torch.int32
    assert s.master[0] is None and s.master[1].dtype == s.master[2].dtype == torch.float32
    s = hb.adamw_state(p)
    assert s.exp_avg_scale is None and s.master is None and not any(t.any() for t in s.exp_avg + s.exp_avg_sq)
    m, v = hb.adamw_moments(s)
    assert all(torch.equal(a, b) for a, b in zip(m + v, s.exp_avg + s.exp_avg_sq)) and m[0] is not s.exp_avg[0]
    strided = torch.ones((4, 6)).t()
    assert hb.adamw_state([strided]).exp_avg[0].stride() == strided.stride() == hb.adamw_state([strided], bits=8).exp_avg[0].stride()


def _shape(hb, rows=100, width=64, hidden=32, experts=4, type=2, activation=0):
    return ctypes.byref(hb._lib.ExpertShape(rows, width, hidden, experts, type, activation))


def _weight(hb, data=A, row=64, expert=2048):
    return ctypes.byref(hb._lib.ExpertWeight(data, row, expert))


def test_expert_entries_refuse(hb):
    lib, bad, ws = hb.load_library(), hb._lib.HB_BAD_ARGUMENT, hb._lib.HB_WORKSPACE
    s, w = _shape(hb), _weight(hb)
    product = [s, A, 64, A, w, A, None]
    gated = [s, A, 64, A, w, w, A, None]
    grad = [s, A, 32, A, 64, A, w, A, A, A, 1 << 40, None]
    gated_grad = [s, A, 32, A, 64, A, w, w, A, A, A, A, 1 << 40, None]
    refused = {
        "no shape": (product, {0: None}), "type": (product, {0: _shape(hb, type=5)}), "rows": (product, {0: _shape(hb, rows=-1)}),
        "too many rows": (product, {0: _shape(hb, rows=2 ** 31)}), "width": (product, {0: _shape(hb, width=0)}),
        "hidden": (gated, {0: _shape(hb, hidden=(1 << 20) + 1)}), "experts": (gated, {0: _shape(hb, experts=0)}),
        "too many experts": (gated, {0: _shape(hb, experts=2049)}), "activation": (gated, {0: _shape(hb, activation=7)}),
        "no offsets": (product, {3: None}), "misaligned offsets": (product, {3: A + 2}), "no x": (product, {1: None}),
        "x off the grid": (_with(product, {0: _shape(hb, rows=1000)}), {1: A + 2}), "x's stride off the grid": (_with(product, {0: _shape(hb, rows=1000)}), {2: 65}),
        "overlapping rows": (_with(product, {0: _shape(hb, rows=1000)}), {2: 56}), "negative stride": (product, {2: -64}),
        "no weight": (product, {4: None}), "weight's address": (product, {4: _weight(hb, data=A + 1)}),
        "weight's rows": (product, {4: _weight(hb, row=56)}), "weight's experts": (product, {4: _weight(hb, expert=-8)}),
        "no out": (product, {5: None}), "out": (product, {5: A + 1}), "no up": (gated, {5: None}), "gated out": (gated, {6: None}),
        "dy off the grid": (grad, {1: A + 8}), "dy's stride": (grad, {2: 36}), "grad x": (grad, {3: None}), "grad weight": (grad, {6: None}),
        "dx": (grad, {7: A + 1}), "dweight": (grad, {8: A + 1}), "dh": (gated_grad, {1: A + 1}), "gated x": (gated_grad, {3: A + 8}),
        "gate": (gated_grad, {6: None}), "up": (gated_grad, {7: _weight(hb, data=A + 8)}), "dup": (gated_grad, {10: A + 1}),
        "gated workspace": (gated_grad, {11: A + 16}), "no workspace": (gated_grad, {11: None}),
    }
    calls = {id(product): lib.hb_expert_product, id(gated): lib.hb_expert_gated, id(grad): lib.hb_expert_product_grad, id(gated_grad): lib.hb_expert_gated_grad}
    for what, (args, change) in refused.items():
        call = calls.get(id(args), lib.hb_expert_product)
        assert call(*_with(args, change)) == bad, what
    assert lib.hb_expert_gated_grad(*_with(gated_grad, {12: 64})) == ws
    split = _shape(hb, rows=1 << 20, experts=1)
    assert lib.hb_expert_product_grad_workspace(split) > 0
    assert lib.hb_expert_product_grad(*_with(grad, {0: split, 10: 64})) == ws
    assert lib.hb_expert_product_grad_workspace(_shape(hb, rows=-1)) == 0 == lib.hb_expert_gated_grad_workspace(None)
    # no rows: nothing to do, whatever the operands
    assert lib.hb_expert_product(*_with(product, {0: _shape(hb, rows=0), 1: None})) == hb._lib.HB_OK
    assert lib.hb_expert_any_grid(_shape(hb, rows=16), 1) and not lib.hb_expert_any_grid(_shape(hb, rows=10 ** 6), 1)
    assert lib.hb_expert_any_grid(_shape(hb, rows=10 ** 6, type=0), 2)


def _with(args, change):
    args = list(args)
    for i, v in change.items():
        args[i] = v
    return args


def test_copies_refuse(hb):
    lib, bad = hb.load_library(), hb._lib.HB_BAD_ARGUMENT

    def call(count=1, source=A, groups=2, rows=3, width=5, to=A, stride=8):
        held = [array("Q", [source]), array("q", [groups]), array("q", [rows]), array("q", [width]), array("q", [15]), array("q", [5]),
                array("Q", [to]), array("q", [stride])]
        return lib.hb_expert_copy(count, *(v.buffer_info()[0] for v in held), None)

    for change in ({"count": 4}, {"count": -1}, {"source": 0}, {"source": A + 1}, {"to": A + 1}, {"groups": -1}, {"rows": -1}, {"width": 0},
                   {"stride": 4}, {"groups": 2 ** 40, "rows": 2 ** 40}):
        assert call(**change) == bad, change
    assert call(rows=0, source=0) == hb._lib.HB_OK


def test_norm_entries_refuse(hb):
    lib, bad, ws = hb.load_library(), hb._lib.HB_BAD_ARGUMENT, hb._lib.HB_WORKSPACE
    norm = [1, A, 64, A, 64, 10, 64, A, 0, 1e-6, A, None, None, A, None]
    for i, v in ((0, 4), (8, 4), (5, -1), (6, 0), (6, 1 << 31), (9, -1.0), (9, float("nan")), (1, None), (1, A + 1), (2, -1), (3, A + 1), (7, None),
                 (7, A + 2), (10, None), (10, A + 1), (11, A), (13, A + 1)):
        assert lib.hb_rms_norm(*_with(norm, {i: v})) == bad, (i, v)
    assert lib.hb_rms_norm(*_with(norm, {10: None, 11: A})) == bad  # codes without scales
    assert lib.hb_rms_norm(*_with(norm, {5: 0, 1: None})) == hb._lib.HB_OK
    back = [A, A, 10, 64, 1, A, None]
    for i, v in ((0, None), (1, None), (2, -1), (3, 0), (4, 9), (5, None), (5, A + 1)):
        assert lib.hb_rows_of_8bit(*_with(back, {i: v})) == bad, (i, v)
    grad = [1, A, 64, A, 64, A, 64, 10, 64, A, 0, 1e-6, A, A, A, 1 << 30, None]
    for i, v in ((0, 4), (1, None), (1, A + 1), (2, -1), (3, None), (5, A + 1), (7, -1), (8, 0), (9, None), (10, 5), (11, -1.0), (12, A + 1),
                 (13, A + 2), (14, None), (14, A + 64)):
        assert lib.hb_rms_norm_grad(*_with(grad, {i: v})) == bad, (i, v)
    assert lib.hb_rms_norm_grad(*_with(grad, {15: 16})) == ws
    assert lib.hb_rms_norm_grad(*_with(grad, {12: None, 13: None})) == hb._lib.HB_OK
    assert lib.hb_rms_norm_grad_workspace(10, 64) > 0 == lib.hb_rms_norm_grad_workspace(-1, 64)


def test_adamw_entries_refuse(hb):
    lib, bad, ws = hb.load_library(), hb._lib.HB_BAD_ARGUMENT, hb._lib.HB_WORKSPACE
    room = lib.hb_adamw_workspace()

    def call(bits=32, address=A, grad=A, state=A, scale=A, master=A, size=1000, type=2, grad_type=2, step=A, work=A, bytes=room, count=1, **rule):
        held = [array("Q", [v]) for v in (address, grad, state, state, scale, scale, master)] + [array("q", [size]), array("i", [type]), array("i", [grad_type])]
        r = hb._lib.AdamWRule(*(rule.get(k, v) for k, v in (("lr", 0.1), ("beta1", 0.9), ("beta2", 0.99), ("eps", 1e-8), ("decay", 0.1), ("max_norm", 1.0),
                                                            ("rate", None), ("norm", None))))
        return lib.hb_adamw_step(count, *(v.buffer_info()[0] for v in held), bits, ctypes.byref(r), step, work, bytes, None)

    for change in ({"bits": 4}, {"count": -1}, {"address": 0}, {"address": A + 1}, {"grad": 0}, {"grad": A + 1}, {"state": 0}, {"state": A + 2},
                   {"master": A + 2}, {"size": -1}, {"type": 3}, {"grad_type": 1}, {"step": None}, {"step": A + 2}, {"work": None}, {"work": A + 8},
                   {"bits": 8, "scale": 0}, {"bits": 8, "scale": A + 2}, {"lr": -1.0}, {"lr": float("nan")}, {"beta1": 1.0}, {"beta2": -0.1},
                   {"eps": -1.0}, {"eps": 1e31}, {"decay": -1.0}, {"norm": A + 2}, {"norm": A, "max_norm": -1.0}, {"rate": A + 1}):
        assert call(**change) == bad, change
    assert call(bytes=room - 1) == ws
    assert lib.hb_adamw_moments(-1, *[None] * 7, None) == bad and lib.hb_adamw_moments(1, *[None] * 7, None) == bad
