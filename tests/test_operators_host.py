"""Routing, lookup and clipping without a GPU: no CPU path, and the host-side checks that come before the
device."""
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
