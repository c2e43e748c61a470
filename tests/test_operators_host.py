"""Routing, lookup and clipping without a GPU: no CPU path, and the host-side checks that come before the
device."""
from array import array

import pytest
import torch


def test_no_cpu_path(hb, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    index, x = torch.zeros((4, 2), dtype=torch.int64), torch.zeros((4, 6))
    plan = hb.RoutePlan(torch.arange(8, dtype=torch.int32), torch.arange(8, dtype=torch.int32).view(4, 2),
                        torch.tensor([0, 8], dtype=torch.int32))
    for call in (lambda: hb.route_plan(index, 3), lambda: hb.route_dispatch(x, plan),
                 lambda: hb.route_combine(torch.zeros((8, 6)), plan), lambda: hb.embedding_lookup(x, index),
                 lambda: hb.embedding_grad(torch.zeros((4, 2, 6)), index, 4), lambda: hb.grad_norm([x]),
                 lambda: hb.clip_grad_norm([x], 1.0)):
        with pytest.raises(hb.HBError, match="requires a CUDA device"):
            call()


def test_plan_properties(hb):
    plan = hb.RoutePlan(torch.arange(6, dtype=torch.int32), torch.arange(6, dtype=torch.int32).view(3, 2),
                        torch.tensor([0, 2, 2, 5], dtype=torch.int32))
    assert (plan.tokens, plan.slots, plan.num_experts, plan.counts.tolist()) == (3, 2, 3, [2, 0, 3])


def test_assignment_of_plan(hb):
    index, weights = hb.assignment_of_plan([1, 0, 1], [0, 2, 3], [0.25, 0.5, 0.25], 3, device="cpu")
    assert index.tolist() == [[2, -1], [0, 3], [-1, -1]] and weights.tolist() == [[1, 0], [0.5, 0.5], [0, 0]]
    index, weights = hb.assignment_of_plan([], [], [], 2, device="cpu")
    assert index.tolist() == [[-1], [-1]] and not weights.any()
    with pytest.raises(ValueError):
        hb.assignment_of_plan([0], [0, 1], [1.0], 2, device="cpu")
    with pytest.raises(ValueError):
        hb.assignment_of_plan([2], [0], [1.0], 2, device="cpu")


def test_workspaces(hb):
    lib = hb.load_library()
    assert lib.hb_index_sort_workspace(1, 64) == 0 and lib.hb_index_sort_workspace(1 << 20, 64) > 0
    assert lib.hb_index_sort_workspace(-1, 64) == 0 and lib.hb_index_sort_workspace(10, 0) == 0
    assert lib.hb_embedding_grad_workspace(1000, 5003, 129) > 0 and lib.hb_clip_workspace(5000) > lib.hb_clip_workspace(5)


def test_entries_refuse_bad_arguments(hb):
    """The C entries check types, sizes, null and misaligned pointers and workspaces before any launch (addresses
    here are made up and never read)."""
    lib, bad, ws = hb.load_library(), hb._lib.HB_BAD_ARGUMENT, hb._lib.HB_WORKSPACE
    a = 1 << 20  # an aligned address
    refused = {
        "index bytes": (lib.hb_index_sort(a, 2, 10, 4, a, a, a, a, 0, None), bad),
        "no bins": (lib.hb_index_sort(a, 4, 10, 0, a, a, a, a, 0, None), bad),
        "too many entries": (lib.hb_index_sort(a, 4, 1 << 31, 4, a, a, a, a, 0, None), bad),
        "no offsets": (lib.hb_index_sort(a, 4, 10, 4, a, a, None, a, 0, None), bad),
        "misaligned index": (lib.hb_index_sort(a + 4, 8, 10, 4, a, a, a, None, 0, None), bad),
        "sort workspace": (lib.hb_index_sort(a, 4, 1 << 20, 4, a, a, a, a, 64, None), ws),
        "misaligned sort workspace": (lib.hb_index_sort(a, 4, 1 << 20, 4, a, a, a, a + 64, 1 << 30, None), bad),
        "element type": (lib.hb_route_dispatch(7, a, 8, 4, 2, 8, a, a, a, None), bad),
        "no slots": (lib.hb_route_dispatch(0, a, 8, 4, 0, 8, a, a, a, None), bad),
        "too many places": (lib.hb_route_dispatch(0, a, 8, 1 << 30, 4, 8, a, a, a, None), bad),
        "null rows": (lib.hb_route_dispatch(0, None, 8, 4, 2, 8, a, a, a, None), bad),
        "misaligned rows": (lib.hb_route_dispatch(0, a + 2, 8, 4, 2, 8, a, a, a, None), bad),
        "weight type": (lib.hb_route_combine(0, a, 8, 4, 2, 8, a, a, a, 9, a, None), bad),
        "misaligned gradient": (lib.hb_route_combine_grad(2, a + 1, 8, a, 8, 4, 2, 8, a, a, a, 0, a, a, None), bad),
        "lookup ids": (lib.hb_embedding_lookup(0, a, 8, 5, 8, a, 3, 4, 1.0, a, None), bad),
        "misaligned ids": (lib.hb_embedding_lookup(0, a, 8, 5, 8, a + 4, 8, 4, 1.0, a, None), bad),
        "gradient type": (lib.hb_embedding_grad(1, a, 8, a, 8, 4, 5, 8, 1.0, 2, a, 0, a, 1 << 30, None), bad),
        "no rows": (lib.hb_embedding_grad(1, a, 8, a, 8, 4, 0, 8, 1.0, 1, a, 0, a, 1 << 30, None), bad),
        "row stride": (lib.hb_embedding_grad(0, a, 1 << 30, a, 8, 4, 5, 8, 1.0, 0, a, 0, a, 1 << 30, None), bad),
        "gradient workspace": (lib.hb_embedding_grad(0, a, 8, a, 8, 4, 5, 8, 1.0, 0, a, 0, a, 8, None), ws),
        "misaligned gradient workspace": (lib.hb_embedding_grad(0, a, 8, a, 8, 4, 5, 8, 1.0, 0, a, 0, a + 8, 1 << 30,
                                                                None), bad),
    }
    for what, (got, want) in refused.items():
        assert got == want, what
    pointers, sizes, types = array("Q", [a]), array("q", [10]), array("i", [0])
    host = [v.buffer_info()[0] for v in (pointers, sizes, types)]
    assert lib.hb_grad_norm(1, *host, a, a, 8, None) == ws
    assert lib.hb_grad_norm(1, *host, a, a + 8, 1 << 20, None) == bad
    assert lib.hb_grad_norm(1, *host, None, a, 1 << 20, None) == bad
    assert lib.hb_clip_grad_norm(1, *host, host[0], host[2], float("nan"), a, a, 1 << 20, None) == bad
    other = array("i", [1])
    assert lib.hb_clip_grad_norm(1, *host, host[0], other.buffer_info()[0], 1.0, a, a, 1 << 20, None) == bad
    pointers[0] = a + 2
    assert lib.hb_grad_norm(1, *host, a, a, 1 << 20, None) == bad
    assert "pointer" in lib.hb_last_error().decode()
