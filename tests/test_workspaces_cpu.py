"""A stream's workspace that grows: what was handed out before stays allocated."""
from __future__ import annotations

import weakref

import pytest
import torch

from aicas_b200 import ops


@pytest.mark.parametrize("get", [ops._workspace, ops._linear_workspace])
def test_replaced_workspaces_stay_alive_and_bounded(monkeypatch, get):
    monkeypatch.setattr(ops, "_WORKSPACES", {})
    monkeypatch.setattr(ops, "_LINEAR_WORKSPACES", {})
    monkeypatch.setattr(ops, "_REPLACED", [], raising=False)
    device, seen = torch.device("cpu"), []
    for size in range(1 << 20, 40 << 20, 1 << 20):  # a graph may have captured any of them
        ws = get(device, 3, size)
        assert ws.numel() >= size and not bool(ws.any()) and get(device, 3, size).data_ptr() == ws.data_ptr()
        seen.append(weakref.ref(ws))
        last = ws.numel()
        del ws
    assert all(r() is not None for r in seen)
    assert sum({r().data_ptr(): r().numel() for r in seen}.values()) <= 2 * last
