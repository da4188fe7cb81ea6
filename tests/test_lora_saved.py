"""What the adapters keep between forward and backward is autograd's: it passes
through saved-tensor hooks, is freed with the graph, and a change of it is seen."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from kernelbench_harbor_b200 import ops
from tests.helpers import w4a16_inputs
from tests.test_lora_apply import inputs


def calls(T):
    c = inputs(T, 256, 128, 8, 3, "bf16", "runs")
    x, q, s, z = w4a16_inputs(T, 256, 128, 64, "bf16", seed=T, device="cuda")
    plan = ops.lora_plan(c["ids"], 3)
    leaves = [c[k].requires_grad_() for k in ("x", "A", "B")]
    return plan, leaves, c["dy"], [lambda x, A, B: ops.lora_apply(c["base"], x, A, B, plan, c["scaling"]),
                                   lambda x, A, B: ops.lora_w4a16(x, q, s, z, 64, A, B, plan, c["scaling"])]


@pytest.mark.gpu
@pytest.mark.parametrize("T", [40, 300])
def test_through_hooks_and_checkpoints(T):
    plan, leaves, dy, forms = calls(T)
    for f in forms:
        want = torch.autograd.grad(f(*leaves), leaves, dy)
        kept = []

        def pack(t):
            kept.append(t.numel() * t.element_size())
            return t.cpu()

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
            y = f(*leaves)
        lo = 4 * T * 16
        assert lo in kept and plan.data.numel() * 4 in kept
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))
        y = checkpoint(f, *leaves, use_reentrant=False)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))


@pytest.mark.gpu
def test_freed_with_the_graph():
    plan, leaves, dy, forms = calls(3000)
    for f in forms:
        y = f(*leaves)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.autograd.grad(y, leaves, dy)
        assert torch.cuda.memory_allocated() <= before - 4 * 3000 * 16


@pytest.mark.gpu
def test_a_changed_plan_is_seen():
    for i in range(2):
        plan, leaves, dy, forms = calls(40)
        y = forms[i](*leaves)
        plan.data.add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, leaves, dy)


@pytest.mark.gpu
def test_a_plan_made_in_inference_mode():
    """Served first, then fitted on: autograd does not save an inference tensor, so it saves a copy."""
    for i in range(2):
        plan, leaves, dy, forms = calls(40)
        want = torch.autograd.grad(forms[i](*leaves), leaves, dy)
        with torch.inference_mode():
            plan.data = plan.data.clone()
        assert plan.data.is_inference()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(forms[i](*leaves), leaves, dy), want))
