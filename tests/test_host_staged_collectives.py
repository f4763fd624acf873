"""Collectives of GPU tensors over a gloo group go through host memory (trainers/averaging.py::on_group)."""
import pytest
import torch
import torch.distributed as dist

from cerberusdet_amd.trainers import averaging


class OnGpu:
    """What on_group asks of a GPU tensor, on the CPU."""

    is_cuda = True

    def __init__(self, values):
        self.held = torch.tensor(values)

    def cpu(self):
        return self.held.clone()

    def copy_(self, t):
        self.held = t.clone()


def doubled(calls):
    def collective(t, group=None, async_op=False, **kw):
        calls.append((type(t), async_op, kw))
        if isinstance(t, torch.Tensor):
            t.mul_(2)
        return "handle" if async_op else None

    return collective


@pytest.mark.parametrize("async_op", [False, True])
def test_gloo_gets_host_memory(monkeypatch, async_op):
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_backend", lambda group=None: "gloo")
    calls, t = [], OnGpu([1.0, 2.0])
    handle = averaging.on_group(doubled(calls), t, async_op=async_op, op=dist.ReduceOp.SUM)
    assert calls == [(torch.Tensor, False, {"op": dist.ReduceOp.SUM})]  # a host tensor, and waited for
    assert t.held.tolist() == [2.0, 4.0]
    assert handle.wait() if async_op else handle is None


def test_other_groups_and_host_tensors_go_as_they_are(monkeypatch):
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_backend", lambda group=None: "nccl")
    calls, t = [], OnGpu([1.0])
    assert averaging.on_group(doubled(calls), t, async_op=True, op=dist.ReduceOp.SUM) == "handle"
    monkeypatch.setattr(dist, "get_backend", lambda group=None: "gloo")
    assert averaging.on_group(doubled(calls), torch.ones(1), async_op=True, op=dist.ReduceOp.SUM) == "handle"
    assert calls == [(OnGpu, True, {"op": dist.ReduceOp.SUM}), (torch.Tensor, True, {"op": dist.ReduceOp.SUM})]


def test_reducer_over_host_staged_units(monkeypatch):
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_world_size", lambda group=None: 2)
    monkeypatch.setattr(dist, "get_backend", lambda group=None: "gloo")
    monkeypatch.setattr(dist, "all_reduce", doubled([]))
    t = OnGpu([3.0])
    t.numel, t.element_size = t.held.numel, t.held.element_size
    r = averaging.GradReducer({0: t}, {0: ["a"]}, ["a"])
    r.reduce_tensor(t, 0)
    r.wait()
    assert t.held.tolist() == [6.0] and r.reduced_bytes == 4 and not r.handles
