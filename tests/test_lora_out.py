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


def forms(c):
    return (lambda out: ops.lora_apply(out, c["x"], c["A"], c["B"], c["ids"], c["scaling"], out=out),
            lambda out: ops.lora_apply(c["base"], c["x"], c["A"], c["B"], c["ids"], c["scaling"], out=out),
            lambda out: ops.lora_expand_add(out, c["x"][:, :8].contiguous(), c["B"], c["ids"].clamp(min=0), out=out))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 300])
def test_what_saved_the_base_sees_the_change(T):
    """base takes no gradient, but an operator before has saved it for its own:
    written over, its backward refuses, as after PyTorch's in-place operators."""
    c = inputs(T, 128, 96, 8, 2, "bf16", "runs")
    for f in forms(c):
        w, base = torch.ones(96, device="cuda").bfloat16().requires_grad_(), c["base"].clone()
        z = base * w
        before = base._version
        assert f(base) is base and base._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()
        # tensors without a version
        with torch.inference_mode():
            base = c["base"].clone()
            want = f(base).clone()
        with torch.no_grad():
            base = c["base"].clone()
            assert torch.equal(f(base), want)
        with torch.inference_mode():
            base = c["base"].clone()
        assert torch.equal(f(base), want)


@pytest.mark.gpu
def test_out_that_asks_for_a_gradient():
    c = inputs(20, 128, 96, 8, 2, "bf16", "runs")
    leaf = torch.zeros_like(c["base"]).requires_grad_()
    for out in (leaf, leaf * 1):
        with pytest.raises(ValueError, match="out cannot be given"):
            ops.lora_apply(c["base"], c["x"], c["A"], c["B"], c["ids"], out=out)
        assert (out == 0).all()
    with torch.no_grad():
        ops.lora_apply(c["base"], c["x"], c["A"], c["B"], c["ids"], out=leaf)
    assert torch.equal(leaf.detach(), ops.lora_apply(c["base"], c["x"], c["A"], c["B"], c["ids"]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("T,D,N,r,L", [(1, 63, 61, 5, 1), (40, 129, 33, 8, 3), (256, 250, 1001, 12, 2), (300, 129, 99, 16, 3),
                                       (700, 333, 1027, 33, 5), (2000, 101, 259, 64, 1), (3000, 257, 65, 4, 700)])
def test_in_place_at_odd_widths(T, D, N, r, L, dtype):
    """Rows that share 16-byte blocks with their neighbours, written while others
    are read: the same bits as beside the base, row by row; dx over the
    projection's likewise."""
    c = inputs(T, D, N, r, L, dtype, "mixed")
    plan = ops.lora_plan(c["ids"], L)
    args = (c["x"], c["A"], c["B"], plan, c["scaling"])
    want = ops.lora_apply(c["base"], *args)
    lo = ops.lora_apply_op(c["base"], c["x"], c["A"], c["B"], c["scaling"], plan.data)[1]
    back = (c["A"], c["B"], c["scaling"], plan.data, lo)
    dx = ops.lora_backward_op(c["x"], c["dy"], c["x"], *back, True, False, False)[0]
    sizes = (T, D, N, r, L, ops._dtype_code(c["x"].dtype))
    for _ in range(5):
        y = c["base"].clone()
        assert ops.lora_apply(y, *args, out=y) is y and torch.equal(y, want)
        g = c["x"].clone()
        ops._lora_grads(sizes, c["x"], c["dy"], g, *back, g, False, False)
        assert torch.equal(g, dx)


@pytest.mark.gpu
def test_out_over_the_plan_or_the_scaling_is_refused():
    """The plan holds row numbers: written over while it is read, it would send a
    kernel anywhere.  Refused on the host, before any launch."""
    c = inputs(10, 64, 8, 8, 16, "fp16", "mixed")
    plan = ops.lora_plan(c["ids"], 16)
    scaling = torch.ones(64, device="cuda")
    for words, kw in ((plan.data, {}), (scaling, {"scaling": scaling[:16]})):
        kept = words.clone()
        out = words.view(torch.float16)[:80].view(10, 8)
        with pytest.raises(ValueError, match="shares memory"):
            ops.lora_apply(c["base"], c["x"], c["A"], c["B"], plan, **kw, out=out)
        assert torch.equal(words, kept)
