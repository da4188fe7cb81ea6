"""Results written over a tensor that autograd knows."""
import pytest
import torch

from kernelbench_harbor_b200 import ops
from tests.test_lora_apply import inputs


@pytest.mark.gpu
def test_module_without_a_gradient_says_so():
    """MultiLoRAW4 adds the adapters over the projection's output.  The projection
    has a gradient, the adapters have none: backward raises, beside another term
    too, and does not return the projection's part alone.  Forward runs."""
    from kernelbench_harbor_b200.modules import MultiLoRAW4
    c = inputs(20, 256, 128, 8, 2, "fp16", "runs")
    q = torch.randint(-8, 8, (256, 128), device="cuda", dtype=torch.int8)
    s, ids = torch.full((2, 128), 0.01, device="cuda").half(), c["ids"].clamp(min=0)
    want = MultiLoRAW4()(c["x"], q, s, c["A"], c["B"], ids)
    x = c["x"].clone().requires_grad_()
    y = MultiLoRAW4()(x, q, s, c["A"], c["B"], ids)
    assert torch.equal(y, want)
    with pytest.raises(RuntimeError, match="lora_expand_add has no gradient"):
        torch.autograd.grad(y.float().sum() + x.float().sum(), x)
    with torch.no_grad():
        assert torch.equal(MultiLoRAW4()(x, q, s, c["A"], c["B"], ids), want)
    # adapters that ask for a gradient beside an input that does not: as ever, none is recorded
    y = MultiLoRAW4()(c["x"], q, s, c["A"].clone().requires_grad_(), c["B"].clone().requires_grad_(), ids)
    assert torch.equal(y, want) and not y.requires_grad
