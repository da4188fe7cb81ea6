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
