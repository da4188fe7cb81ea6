"""Gradients of gradients: right, or refused; never dropped without a word.  And
the operators as traced programs see them."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from kernelbench_harbor_b200 import ops
from tests.helpers import torch_dequant_fp32, w4a16_inputs


# ---------------------------------------------------------------- the frozen projection
@pytest.mark.gpu
@pytest.mark.parametrize("M,dtype", [(5, "bf16"), (40, "fp16"), (200, "bf16")])
def test_second_gradient_through_the_projection(M, dtype):
    """L = sum(g^2) + sum(x), g the gradient of sum(y^2) / 2 in x, y = x . W:
    dL/dx = 2 W W^T W W^T x + 1, with the roundings of y, g, 2 g (exact), its
    products and the last counted: each at most u of its value, and the weight's
    as the kernels hold it."""
    x, q, s, z = w4a16_inputs(M, 256, 128, 64, dtype, seed=M, device="cuda")
    x.requires_grad_()
    u = torch.finfo(x.dtype).eps / 2
    y = ops.w4a16_gemm(x, q, s, z, 64)
    (g,) = torch.autograd.grad(0.5 * y.square().sum(dtype=torch.float32), x, create_graph=True)
    assert g.requires_grad
    (d,) = torch.autograd.grad(g.square().sum(dtype=torch.float32) + x.sum(dtype=torch.float32), x)
    w = torch_dequant_fp32(q, s, z, 64).double()
    ww, aa = w @ w.t(), w.abs() @ w.abs().t()
    xd = x.detach().double()
    want = 2 * xd @ ww @ ww + 1
    # four passes through the weight (u each for its rounding), and as many results rounded
    mag = 2 * xd.abs() @ aa @ aa
    assert ((d.double() - want).abs() <= 10 * u * mag + 2 * u * want.abs()).all()
    assert float(want.abs().mean()) > 4  # the second term is a small part


@pytest.mark.gpu
def test_gradient_of_the_input_gradient():
    """w4a16_dgrad is linear in dy: its gradient is w4a16_gemm, bit for bit."""
    _, q, s, z = w4a16_inputs(1, 256, 128, 64, "fp16", seed=3, device="cuda")
    dy = torch.randn(30, 128, device="cuda").half().requires_grad_()
    v = torch.randn(30, 256, device="cuda").half()
    dx = ops.w4a16_dgrad(dy, q, s, z, 64)
    assert torch.equal(dx, ops.w4a16_dgrad(dy.detach(), q, s, z, 64))
    assert torch.equal(torch.autograd.grad(dx, dy, v)[0], ops.w4a16_gemm(v, q, s, z, 64))
    with pytest.raises(RuntimeError, match="frozen"):
        ops.w4a16_dgrad(dy, q, s.clone().requires_grad_(), z, 64).sum().backward()


def test_projection_on_fake_tensors():
    with FakeTensorMode():
        x, q = torch.empty(5, 256, dtype=torch.float16).requires_grad_(), torch.empty(256, 16, dtype=torch.int32)
        s = torch.empty(4, 128, dtype=torch.float16)
        y = ops.w4a16_gemm(x, q, s, s, 64)
        (dx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        (ddx,) = torch.autograd.grad(dx.square().sum(), x)
        assert dx.shape == ddx.shape == x.shape and dx.requires_grad and ddx.dtype == torch.float16
        assert ops.w4a16_dgrad(y.detach(), q, s, s, 64).shape == (5, 256)


@pytest.mark.gpu
def test_projection_compiled():
    x, q, s, z = w4a16_inputs(40, 256, 128, 64, "bf16", seed=1, device="cuda")
    x.requires_grad_()
    v = torch.randn(40, 128, device="cuda").bfloat16()

    def loss(x):
        return (ops.w4a16_gemm(x, q, s, z, 64) * v).float().sum()

    (want,) = torch.autograd.grad(loss(x), x)
    (got,) = torch.autograd.grad(torch.compile(loss, backend="aot_eager", fullgraph=True)(x), x)
    assert torch.equal(got, want)
    dgrad = torch.compile(lambda d: ops.w4a16_dgrad(d, q, s, z, 64), backend="aot_eager", fullgraph=True)
    assert torch.equal(dgrad(v), ops.w4a16_dgrad(v, q, s, z, 64))


# ---------------------------------------------------------------- adapters and balance loss: refused
def adapters(T, seed=0):
    g = torch.Generator().manual_seed(seed + T)
    n = lambda *s: (torch.randn(*s, generator=g) * 0.3).half().cuda()  # noqa: E731
    return dict(base=n(T, 64), x=n(T, 128), A=n(2, 128, 8), B=n(2, 8, 64)), torch.randint(-1, 2, (T,), generator=g).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("T", [20, 300])
def test_adapter_gradients_refuse_a_second_one(T, strided):
    """With a constant upstream gradient dx depends on A and B, dA on x and B, dB on
    x and A: a term built on one of them is refused, beside another term too.
    Where nothing that it depends on asks for a gradient, it is a constant."""
    c, ids = adapters(T)
    if strided:  # what autograd has to follow through a copy
        c["x"] = torch.cat([c["x"], c["x"]], dim=1)[:, :128]
        c["A"], c["B"] = c["A"].transpose(1, 2).contiguous().transpose(1, 2), c["B"].transpose(1, 2).contiguous().transpose(1, 2)
    v = torch.randn(T, 64, device="cuda").half()
    for of in ("x", "A", "B"):
        for on in ("x", "A", "B"):
            leaf = {k: t.detach().clone(memory_format=torch.preserve_format).requires_grad_(k in (of, on)) for k, t in c.items()}
            y = ops.lora_apply(leaf["base"], leaf["x"], leaf["A"], leaf["B"], ids)
            (g,) = torch.autograd.grad(y, leaf[of], v, create_graph=True)
            loss = g.float().square().sum() + leaf[on].float().sum()
            if of == on:
                assert not g.requires_grad and torch.equal(torch.autograd.grad(loss, leaf[on])[0], torch.ones_like(leaf[on]))
            else:
                with pytest.raises(RuntimeError, match="lora_backward"):
                    torch.autograd.grad(loss, leaf[on])
    # a gradient of y that depends on y
    x = c["x"].detach().clone().requires_grad_()
    y = ops.lora_apply(c["base"], x, c["A"], c["B"], ids)
    (g,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="lora_backward"):
        (g.float().square().sum() + x.float().sum()).backward()
    assert torch.equal(g.detach(), torch.autograd.grad(ops.lora_apply(c["base"], x, c["A"], c["B"], ids).float().square().sum(), x)[0])


@pytest.mark.gpu
def test_gradient_of_the_base_has_a_gradient():
    """base's gradient is y's own: differentiated as often as y."""
    c, ids = adapters(40)
    base, A = c["base"].requires_grad_(), c["A"].requires_grad_()
    y = ops.lora_apply(base, c["x"], A, c["B"], ids)
    (g,) = torch.autograd.grad(y.float().square().sum(), base, create_graph=True)
    got = torch.autograd.grad(g.float().square().sum(), (base, A))
    y = ops.lora_apply(base, c["x"], A, c["B"], ids)
    want = torch.autograd.grad((2 * y).float().square().sum(), (base, A))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 300])
def test_adapted_projection_refuses_a_second_gradient(T):
    x, q, s, z = w4a16_inputs(T, 128, 64, 64, "fp16", seed=T, device="cuda")
    c, ids = adapters(T)
    v = torch.randn(T, 64, device="cuda").half()
    for of, on in (("x", "A"), ("A", "x"), ("B", "A"), ("x", "B")):
        leaf = {k: t.clone().requires_grad_(k in (of, on)) for k, t in dict(c, x=x).items()}
        y = ops.lora_w4a16(leaf["x"], q, s, z, 64, leaf["A"], leaf["B"], ids)
        (g,) = torch.autograd.grad(y, leaf[of], v, create_graph=True)
        with pytest.raises(RuntimeError, match="lora_backward"):
            torch.autograd.grad(g.float().square().sum() + leaf[on].float().sum(), leaf[on])
        y = ops.lora_w4a16(leaf["x"], q, s, z, 64, leaf["A"], leaf["B"], ids)
        assert torch.equal(g.detach(), torch.autograd.grad(y, leaf[of], v)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("strided", [False, True])
def test_balance_gradient_refuses_a_second_one(strided):
    lg = torch.randn(50, 8, device="cuda")
    lg = (torch.cat([lg, lg], dim=1)[:, :8] if strided else lg).requires_grad_()
    topi = torch.topk(lg.detach(), 2, dim=1).indices
    loss, _ = ops.moe_balance_loss(lg, topi)
    (d,) = torch.autograd.grad(loss, lg, create_graph=True)
    with pytest.raises(RuntimeError, match="moe_balance_grad"):
        (d.square().sum() + lg.sum()).backward()
    loss, _ = ops.moe_balance_loss(lg, topi)
    assert torch.equal(d.detach(), torch.autograd.grad(loss, lg)[0])


@pytest.mark.gpu
def test_registered_operators_refuse_what_does_not_fit():
    c, ids = adapters(40)
    plan = ops.lora_plan(ids, 2).data
    lo = torch.zeros(40, 16, device="cuda")
    dy = torch.zeros(40, 64, device="cuda").half()
    ok = dict(x=c["x"], dy=dy, base=None, A=c["A"], B=c["B"], scaling=None, plan=plan, lo=lo, want_x=True, want_A=True, want_B=True)
    ops.lora_backward_op(**ok)
    for bad in (dict(dy=dy[:, :32]), dict(dy=dy.float()), dict(A=c["A"][:1]), dict(plan=plan[:40]), dict(plan=plan.long()),
                dict(lo=lo[:, :8]), dict(base=dy), dict(scaling=torch.ones(1, device="cuda")), dict(lo=lo.cpu())):
        with pytest.raises((ValueError, TypeError)):
            ops.lora_backward_op(**{**ok, **bad})
    lg, coef, one = torch.zeros(4, 8, device="cuda"), torch.zeros(8, device="cuda"), torch.ones((), device="cuda")
    ops.moe_balance_grad_op(lg, None, coef, one)
    for args in ((lg.double(), None, coef, one), (lg, None, coef[:7], one), (lg, None, coef, one.half()),
                 (lg, torch.ones(3, dtype=torch.bool, device="cuda"), coef, one), (lg, None, coef, one.cpu())):
        with pytest.raises((ValueError, TypeError)):
            ops.moe_balance_grad_op(*args)


# ---------------------------------------------------------------- forward mode: refused
def test_tangents_are_refused():
    """On any device: the check comes first, and a tensor without a tangent goes on."""
    import torch.autograd.forward_ad as fw
    z = torch.zeros
    ids, plain = z(4, dtype=torch.int64), dict(base=z(4, 8), x=z(4, 8), A=z(2, 8, 4), B=z(2, 4, 8))
    q, s = z(8, 1, dtype=torch.int32), z(1, 8)
    with fw.dual_level():
        dual = {k: fw.make_dual(t, torch.ones_like(t)) for k, t in plain.items()}
        for k in plain:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ops.lora_apply(**{**plain, k: dual[k]}, plan=ids)
        for k in ("x", "A", "B"):
            a = {**plain, k: dual[k]}
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ops.lora_w4a16(a["x"], q, s, s, 8, a["A"], a["B"], ids)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.w4a16_dgrad(dual["x"], q, s, s, 8)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.w4a16_gemm(dual["x"], q, s, s, 8)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.moe_balance_loss(dual["x"], z(4, 2, dtype=torch.int32))
        with pytest.raises(RuntimeError, match="CUDA"):  # no tangent: on to the next check
            ops.lora_apply(**plain, plan=ids)


@pytest.mark.gpu
def test_tangent_of_the_base_is_refused():
    import torch.autograd.forward_ad as fw
    c, ids = adapters(20)
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.lora_apply(fw.make_dual(c["base"], c["base"]), c["x"], c["A"], c["B"], ids)
        lg = fw.make_dual(torch.zeros(4, 8, device="cuda"), torch.ones(4, 8, device="cuda"))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.moe_balance_loss(lg, torch.zeros(4, 2, dtype=torch.int32, device="cuda"))
        ops.lora_apply(c["base"], c["x"], c["A"], c["B"], ids)  # no tangent: as ever
