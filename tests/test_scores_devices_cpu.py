"""Launches of the score operators for tensors of a device that is not the current one: on that device and its stream, and without tickets
(which belong to a stream of the current device)."""
import contextlib

import pytest
import torch

import helpers as H  # noqa: F401  (puts the repo root on sys.path)
from vitta_amd import _lib, ops


def test_a_launch_goes_to_the_tensors_device(monkeypatch):
    current, seen = [0], []

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        try:
            yield
        finally:
            current[0] = before
    monkeypatch.setattr(ops, "_current_device", lambda: current[0])
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 100 + index)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setitem(ops._entry_points, "a launch", lambda *args: seen.append((current[0], args)) or 0)
    monkeypatch.setitem(ops._entry_points, "a refused one", lambda *args: -1)
    ops._call("a launch", 0, 7)
    ops._call("a launch", 3, 8)
    assert seen == [(0, (7, 100)), (3, (8, 103))] and current == [0]
    with pytest.raises(_lib.VittaHipError, match="a refused one"):
        ops._call("a refused one", 3)
    assert current == [0]


def test_tickets_belong_to_streams_of_the_current_device(monkeypatch):
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 5)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(ops, "_score_tickets", {})
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 1)
    m = torch.zeros(1, 131072, dtype=torch.bfloat16)
    ws, n, tickets = ops._score_workspace(m, 1, 131072, 1, 0)
    assert n > 0 and ws.numel() == n and tickets is None and ops._score_tickets == {}
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    assert ops._score_workspace(m, 1, 131072, 1, 0)[2] == ops._score_tickets[0, 5].data_ptr()
    assert ops._score_workspace(m, 1, 131072, 1, 0)[2] == ops._score_tickets[0, 5].data_ptr()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert ops._score_workspace(m, 1, 131072, 1, 0)[2] is None
