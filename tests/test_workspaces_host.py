"""The cached workspaces of ops, on the CPU: what a CUDA graph captured earlier may still name stays allocated."""
import weakref

import pytest
import torch

from comfy_ui_gfx906_tools_b200 import ops


@pytest.mark.parametrize("get,cache", [(ops._workspace, "_workspaces"), (ops._exact_workspace, "_exact_workspaces")])
def test_an_outgrown_workspace_stays_allocated(monkeypatch, get, cache):
    monkeypatch.setattr(ops, cache, {})
    monkeypatch.setattr(ops, "_retired", [])
    cpu = torch.device("cpu")
    first = get(cpu, 7, 1000)
    assert first.numel() == 1 << 20 and get(cpu, 7, 1 << 20) is first and get(cpu, 8, 1000) is not first
    alive, at = weakref.ref(first), first.data_ptr()
    del first
    sizes = [1 << 20]
    for need in ((1 << 20) + 1, 5 << 20, (5 << 20) + 1):
        ws = get(cpu, 7, need)
        assert ws.numel() >= need and ws.numel() >= 2 * sizes[-1] and get(cpu, 7, 1000) is ws
        sizes.append(ws.numel())
        del ws
    assert alive() is not None and alive().data_ptr() == at
    assert sum(sizes) < 2 * sizes[-1]


def test_outgrown_workspaces_are_rearmed_too(monkeypatch):
    """After a wait gave up, a graph's counters have to be zero again as well."""
    monkeypatch.setattr(ops, "_workspaces", {})
    monkeypatch.setattr(ops, "_retired", [])
    cpu = torch.device("cpu")
    a = ops._workspace(cpu, 7, 1000)
    b = ops._workspace(cpu, 7, 2 << 20)
    assert int(a.max()) == 0 and int(b.max()) == 0
    for ws in (a, b):
        ws.fill_(1)
    ops._rearm_workspaces(cpu)
    assert int(a.max()) == 0 and int(b.max()) == 0
