"""The adapter operators and the balance loss as traced programs see them: fake
tensors, export, torch.compile; and under a dispatch mode."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

from kernelbench_harbor_b200 import _lib, ops
from kernelbench_harbor_b200.modules import LoRAW4A16Linear, MoEBalanceLoss
from tests.helpers import w4a16_inputs
from tests.test_lora_apply import inputs


def test_sizes_of_the_fake_forms():
    import kernelbench_harbor_b200 as pkg
    pkg.build()
    L = _lib.lib()
    for T in (0, 1, 15, 16, 17, 127, 128, 129, 1000, 1 << 20):
        for n in (1, 2, 7, 64, 1023):
            assert 4 * ops._plan_words(T, n) == L.b200q_lora_plan_bytes(T, n)
        for r in (1, 16, 17, 32, 33, 64):
            x, A, plan = torch.empty(T, 1), torch.empty(1, 1, r), torch.empty(1, dtype=torch.int32)
            if T < 2000:
                assert 4 * ops._lo_words(x, A, plan).numel() == L.b200q_lora_mid_bytes(T, r)


class Layer(torch.nn.Module):
    def forward(self, x, q, s, z, A, B, ids, scaling, router):
        plan = ops.lora_plan(ids, A.shape[0])
        y = LoRAW4A16Linear()(x, q, s, z, A, B, plan, scaling)
        y = ops.lora_apply(y, x, A, B, plan)
        logits = x @ router
        loss, counts = MoEBalanceLoss()(logits, ops.moe_route(logits.detach())[0], ids >= 0)
        return y, loss, counts


def on_fakes(T=40):
    h = dict(dtype=torch.float16, device="cuda")
    return (torch.empty(T, 256, **h), torch.empty(256, 16, dtype=torch.int32, device="cuda"), torch.empty(4, 128, **h),
            torch.empty(4, 128, **h), torch.empty(3, 256, 8, **h), torch.empty(3, 8, 128, **h),
            torch.empty(T, dtype=torch.int64, device="cuda"), torch.empty(3, device="cuda"), torch.empty(256, 8, **h))


def test_on_fake_tensors():
    with FakeTensorMode():
        args = on_fakes()
        y, loss, counts = Layer()(*args)
        assert y.shape == (40, 128) and y.dtype == torch.float16 and y.device == args[0].device
        assert loss.shape == () and loss.dtype == torch.float32 and counts.shape == (8,) and counts.dtype == torch.int32
        x, A, B, plan = args[0], args[4], args[5], ops.lora_plan(args[6], 3)
        assert ops.lora_apply(y, x, A, B, plan, out=y) is y
        grads = ops.lora_backward_op(x, y, None, A, B, None, plan.data, ops._lo_words(x, A, plan.data), True, False, True)
        assert [tuple(g.shape) for g in grads] == [(40, 256), (0,), (3, 8, 128)]
        lg = torch.empty(40, 8, device="cuda", dtype=torch.bfloat16)
        assert ops.moe_balance_grad_op(lg, None, torch.empty(8, device="cuda"), loss).dtype == torch.bfloat16


def test_exported():
    with FakeTensorMode():
        program = torch.export.export(Layer(), on_fakes())
    calls = {n.target.name() for n in program.graph.nodes if n.op == "call_function" and hasattr(n.target, "name")}
    assert {"b200q::lora_plan", "b200q::lora_w4a16", "b200q::lora_apply", "b200q::moe_balance"} <= calls


def setup(T, dtype="bf16"):
    x, q, s, z = w4a16_inputs(T, 256, 128, 64, dtype, seed=T, device="cuda")
    c = inputs(T, 256, 128, 8, 3, dtype, "runs")
    router = (torch.randn(256, 8, device="cuda") * 0.1).to(x.dtype)
    return [x, q, s, z, c["A"], c["B"], c["ids"], c["scaling"], router]


@pytest.mark.gpu
@pytest.mark.parametrize("dynamic", [False, True])
def test_compiled_forward_and_backward(dynamic):
    """The same bits compiled as eagerly, with gradients."""
    step = torch.compile(Layer(), backend="aot_eager", fullgraph=True, dynamic=dynamic)
    for T in (40, 300):
        args = setup(T)
        leaves = [args[i].requires_grad_() for i in (0, 4, 5, 8)]
        v = torch.randn(T, 128, device="cuda").bfloat16()

        def run(f):
            y, loss, counts = f(*args)
            return (y, loss, counts, *torch.autograd.grad((y, loss), leaves, (v, torch.full_like(loss, 16.0))))

        for a, b in zip(run(step), run(Layer())):
            assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)
        with torch.no_grad():
            assert all(torch.equal(a, b) for a, b in zip(step(*args), Layer()(*args)))


@pytest.mark.gpu
def test_under_a_dispatch_mode():
    """A mode sees the calls, and they give the same bits."""
    class Names(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = set()

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.add(func.name())
            return func(*args, **(kwargs or {}))

    args = setup(40)
    leaves = [args[i].requires_grad_() for i in (0, 4, 5, 8)]

    def run():
        y, loss, counts = Layer()(*args)
        return (y, loss, counts, *torch.autograd.grad(y.float().sum() + loss, leaves))

    want = run()
    with Names():  # backward behind the mode
        y, loss, counts = Layer()(*args)
    behind = (y, loss, counts, *torch.autograd.grad(y.float().sum() + loss, leaves))
    with Names() as names:
        got = run()
    assert all(torch.equal(a, b) for a, b in zip(behind, want))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert {"b200q::lora_plan", "b200q::lora_w4a16", "b200q::lora_apply", "b200q::lora_backward", "b200q::w4a16_dgrad",
            "b200q::moe_balance", "b200q::moe_balance_grad"} <= names.seen


@pytest.mark.gpu
def test_in_place_while_traced():
    x, q, s, z, A, B, ids, scaling, _ = setup(40)
    base = ops.w4a16_gemm(x, q, s, z, 64)
    want = ops.lora_apply(base, x, A, B, ids, scaling)

    def f(base):
        return ops.lora_apply(base, x, A, B, ids, scaling, out=base)

    got = base.clone()
    torch.compile(f, backend="aot_eager", fullgraph=True)(got)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_a_plan_handed_to_a_compiled_program():
    x, q, s, z, A, B, ids, scaling, _ = setup(40)
    plan = ops.lora_plan(ids, 3)
    f = torch.compile(lambda x, plan: ops.lora_w4a16(x, q, s, z, 64, A, B, plan, scaling), backend="aot_eager", fullgraph=True)
    assert torch.equal(f(x, plan), ops.lora_w4a16(x, q, s, z, 64, A, B, plan, scaling))
    other = ops.lora_plan(ids.flip(0), 3)
    assert torch.equal(f(x, other), ops.lora_w4a16(x, q, s, z, 64, A, B, other, scaling))
