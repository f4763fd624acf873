"""Every tensor collective of the package goes through on_group, which keeps device tensors away from gloo."""
import ast
from pathlib import Path

import pytest
import torch
import torch.distributed as dist

from cerberusdet_amd.trainers import averaging
from test_host_staged_collectives import OnGpu

PACKAGE = Path(averaging.__file__).resolve().parents[1]
OF_TENSORS = {"all_reduce", "broadcast", "reduce", "all_gather", "all_gather_into_tensor", "reduce_scatter", "reduce_scatter_tensor", "all_to_all", "all_to_all_single", "gather",
              "scatter", "send", "recv", "isend", "irecv"}


@pytest.mark.parametrize("path", sorted(PACKAGE.rglob("*.py")), ids=lambda p: str(p.relative_to(PACKAGE)))
def test_no_tensor_collective_is_called_directly(path):
    calls = [n for n in ast.walk(ast.parse(path.read_text())) if isinstance(n, ast.Call) and isinstance(n.func, ast.Attribute)]
    direct = [f"{path.name}:{n.lineno} dist.{n.func.attr}" for n in calls
              if n.func.attr in OF_TENSORS and isinstance(n.func.value, ast.Name) and n.func.value.id in ("dist", "distributed")]
    assert not direct


def test_broadcast_of_a_device_tensor_over_gloo(monkeypatch):
    """What train.py sends at its start and its stop: the values arrive from host memory, under the caller's src."""
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_backend", lambda group=None: "gloo")
    seen = []

    def broadcast(t, src=None, group=None):
        seen.append((type(t), src))
        t.fill_(7)

    flag = OnGpu([0])
    assert averaging.on_group(broadcast, flag, src=0) is None
    assert seen == [(torch.Tensor, 0)] and flag.held.tolist() == [7]
