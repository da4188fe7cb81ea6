"""Workspaces beside graph captures."""
import gc
import weakref

import pytest
import torch

from kernelbench_harbor_b200 import ops


@pytest.fixture
def on_cpu(monkeypatch):
    """The bookkeeping alone: buffers on the host, a stream by number."""
    monkeypatch.setattr(ops, "_stream_ptr", lambda device: 7)
    monkeypatch.setattr(ops, "_ws", {})
    monkeypatch.setattr(ops, "_ws_outgrown", [])
    return None, None, lambda n: ops.workspace(torch.device("cpu", 0), n)


def test_outgrown_workspaces_stay(on_cpu):
    """A captured graph holds the address of the one that it was captured with."""
    _, _, ws = on_cpu
    first = ws(256)
    assert ws(1024) is first
    ref, at = weakref.ref(first), first.data_ptr()
    more = ws(1 << 20)
    del first
    gc.collect()
    assert more.numel() >= 1 << 20 and ref() is not None and ref().data_ptr() == at and more.data_ptr() != at
    ops.reset_workspaces()
    gc.collect()
    assert ref() is None
