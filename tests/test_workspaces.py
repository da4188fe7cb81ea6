"""Workspaces beside graph captures: graphs replayed in any order, and calls that
need more room later."""
import gc
import weakref

import pytest
import torch

from kernelbench_harbor_b200 import _lib, ops
from tests.helpers import w4a16_inputs


class FakeLib:
    capture = 0

    def b200q_capture_id(self, stream):
        return self.capture


@pytest.fixture
def on_cpu(monkeypatch):
    """The bookkeeping alone: buffers on the host, a stream and captures by number."""
    lib, stream = FakeLib(), [7]
    monkeypatch.setattr(_lib, "_lib", lib)
    monkeypatch.setattr(ops, "_stream_ptr", lambda device: stream[0])
    for name in ("_ws", "_ws_captured"):
        monkeypatch.setattr(ops, name, {})
    monkeypatch.setattr(ops, "_ws_outgrown", [])
    return lib, stream, lambda n: ops.workspace(torch.device("cpu", 0), n)


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


def test_zeroed_in_every_capture(on_cpu):
    lib, stream, ws = on_cpu
    lib.capture = 1
    a = ws(256)
    a.fill_(5)
    assert ws(256) is a and int(a[0]) == 5  # once a capture
    lib.capture = 2
    assert ws(256) is a and int(a.count_nonzero()) == 0
    a.fill_(5)
    stream[0] = 8  # another stream has its own
    assert ws(256) is not a
    stream[0] = 7
    lib.capture = 0
    b = ws(256)  # outside: not what waits for its graph
    assert b is not a and int(b.count_nonzero()) == 0
    b.fill_(5)
    lib.capture = 3
    assert ws(256) is b and int(b[0]) == 5  # zeroed when it was made; kernels keep it so
    assert any(t is a for t in ops._ws_outgrown)


@pytest.mark.gpu
def test_capture_id():
    lib, s = _lib.lib(), torch.cuda.Stream()
    assert lib.b200q_capture_id(None) == lib.b200q_capture_id(s.cuda_stream) == 0
    ids, x = [], torch.zeros(4, device="cuda")
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            x.add_(1)
            ids.append(lib.b200q_capture_id(s.cuda_stream))
    assert 0 not in ids and ids[0] != ids[1] and lib.b200q_capture_id(s.cuda_stream) == 0


@pytest.mark.gpu
def test_graphs_replayed_in_another_order():
    """Two decode steps, both captured on a stream that has run nothing: the
    second one's workspace is in order before the first was ever replayed."""
    s = torch.cuda.Stream()
    graphs = []
    for seed in (1, 2):
        x, q, sc, z = w4a16_inputs(8, 4096, 1024, 128, "fp16", seed=seed, device="cuda")
        want = ops.w4a16_gemm(x, q, sc, z, 128)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = ops.w4a16_gemm(x, q, sc, z, 128)
        graphs.append((g, y, want, (x, q, sc, z)))
    # the memory as another owner may have left it
    with torch.cuda.stream(s):
        key = (torch.cuda.current_device(), s.cuda_stream)
        ops._ws[key].fill_(1)
    s.synchronize()
    for i in (1, 0, 1, 1, 0):
        g, y, want, _ = graphs[i]
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    # eager calls on that stream take a workspace of their own
    with torch.cuda.stream(s):
        assert torch.equal(ops.w4a16_gemm(*graphs[0][3], 128), graphs[0][2])
        assert ops.device_status() == 0
