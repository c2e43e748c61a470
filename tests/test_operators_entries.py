"""Refusals of the C entries of the routing, lookup and clipping operators, and of what else of them needs no GPU
(addresses are made up and never read)."""
from array import array

import pytest

A = 1 << 20  # an aligned address


def test_misaligned_arrays(hb):
    """Kernels read and write whole elements: an address between them is refused before any launch."""
    lib, bad = hb.load_library(), hb._lib.HB_BAD_ARGUMENT
    ws = lib.hb_index_sort_workspace(10, 4)
    for off in (1, 2, 3):
        sort = [A, 4, 10, 4, A, A, A, A, ws, None]
        for at in (0, 4, 5, 6):
            args = list(sort)
            args[at] += off
            assert lib.hb_index_sort(*args) == bad, (off, at)
        for weight_type in (0, 1, 2):
            dispatch = [0, A, 8, 4, 2, 8, A, A, A, None]
            combine = [0, A, 8, 4, 2, 8, A, A, A, weight_type, A, None]
            grad = [0, A, 8, A, 8, 4, 2, 8, A, A, A, weight_type, A, A, None]
            whole = weight_type != 0 and off == 2  # 16-bit weights lie on 2 bytes
            for call, args, places in ((lib.hb_route_dispatch, dispatch, (6, 7)),
                                       (lib.hb_route_combine, combine, (6, 7) + (() if whole else (8,))),
                                       (lib.hb_route_combine_grad, grad, (8, 9) + (() if whole else (10, 13)))):
                for at in places:
                    wrong = list(args)
                    wrong[at] += off
                    assert call(*wrong) == bad, (call.__name__, off, at)
        pointers, sizes, types = array("Q", [A]), array("q", [10]), array("i", [0])
        host = [v.buffer_info()[0] for v in (pointers, sizes, types)]
        room = lib.hb_clip_workspace(1)
        assert lib.hb_grad_norm(1, *host, A + off, A, room, None) == bad
        assert lib.hb_clip_grad_norm(1, *host, host[0], host[2], 1.0, A + off, A, room, None) == bad


def test_plans_that_are_no_assignment(hb):
    """A mass that is no number, or an expert that is none, is refused, where it was left out of the token's shares."""
    inf, nan = float("inf"), float("nan")
    for rows, cols, mass in (([0, 1], [-1, 0], [0.5, 0.5]), ([0, 1], [0, 2 ** 31], [0.5, 0.5]), ([0, 1], [0, 2 ** 32], [0.5, 0.5]),
                             ([0, 0], [0, 1], [0.5, nan]), ([0, 0], [0, 1], [0.5, inf])):
        with pytest.raises(ValueError):
            hb.assignment_of_plan(rows, cols, mass, 2, device="cpu")
    # an edge without mass is no entry, whatever its ends
    index, weights = hb.assignment_of_plan([0, -1, 1], [0, -1, 2 ** 40], [0.5, 0.0, 0.0], 2, device="cpu")
    assert index.tolist() == [[0], [-1]] and weights.tolist() == [[1], [0]]
