"""Tensors on a device that is not the current one."""
import pytest
import torch

from kernelbench_harbor_b200 import _lib, ops
from tests.helpers import w4a16_inputs
from tests.test_lora_apply import inputs


class Watched:
    """The library, with the calls that launch noted together with the device that was made current for them."""

    def __init__(self, lib, inside):
        self.lib, self.inside, self.calls = lib, inside, []

    def __getattr__(self, name):
        fn = getattr(self.lib, name)
        if name.endswith("_bytes") or name.endswith("_error"):
            return fn

        def call(*args):
            self.calls.append((name, self.inside[-1] if self.inside else None))
            return fn(*args)

        return call


@pytest.mark.gpu
@pytest.mark.parametrize("T", [10, 300])
def test_every_launch_is_made_on_the_tensors_device(T, monkeypatch):
    """One GPU is enough: each call of the library has to come from within the
    context that makes its tensors' device the current one."""
    x, q, s, z = w4a16_inputs(T, 256, 128, 64, "bf16", seed=T, device="cuda")
    c = inputs(T, 256, 128, 8, 3, "bf16", "runs")
    lg = torch.randn(T, 8, device="cuda").requires_grad_()
    topi = torch.topk(lg.detach(), 2, dim=1).indices.int()
    inside, real = [], ops._device

    class Entered:
        def __init__(self, device):
            self.device, self.ctx = device, real(device)

        def __enter__(self):
            inside.append(self.device)
            return self.ctx.__enter__()

        def __exit__(self, *exc):
            inside.pop()
            return self.ctx.__exit__(*exc)

    watched = Watched(_lib.lib(), inside)
    monkeypatch.setattr(ops, "_device", Entered)
    monkeypatch.setattr(_lib, "_lib", watched)
    leaves = [t.clone().requires_grad_() for t in (x, c["A"], c["B"])]
    plan = ops.lora_plan(c["ids"], 3)
    with torch.no_grad():
        y = ops.lora_w4a16(x, q, s, z, 64, c["A"], c["B"], plan, c["scaling"])
        ops.lora_apply(y, x, c["A"], c["B"], plan, out=y)
    torch.autograd.grad(ops.lora_w4a16(leaves[0], q, s, z, 64, *leaves[1:], plan), leaves, c["dy"])
    torch.autograd.grad(ops.lora_apply(c["base"], *leaves, plan), leaves, c["dy"])
    torch.autograd.grad(ops.w4a16_gemm(leaves[0], q, s, z, 64), leaves[0], c["dy"])
    torch.autograd.grad(ops.moe_balance_loss(lg, topi)[0], lg)
    names = {n for n, _ in watched.calls}
    assert {"b200q_" + n for n in ("lora_plan", "lora_apply", "lora_backward", "w4a16_gemm", "w4a16_dgrad", "moe_balance",
                                   "moe_balance_grad")} <= names
    assert [n for n, d in watched.calls if d != x.device] == []


@pytest.mark.gpu
def test_a_device_without_an_index_is_the_current_one():
    cuda, numbered = torch.device("cuda"), torch.device("cuda", torch.cuda.current_device())
    assert ops.workspace(cuda, 256) is ops.workspace(numbered, 256)
    assert ops.device_status(cuda) == 0
    ops.lora_plan(torch.tensor([0, 5, -1], device="cuda"), 2)
    assert ops.device_status(cuda) & 2 and ops.device_status(numbered) == 0
