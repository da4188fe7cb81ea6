"""Input gradient of the frozen W4A16 projection, dx = dy . dequant(W)^T,
against float64."""
import pytest
import torch

from kernelbench_harbor_b200 import _lib, ops
from tests.helpers import tdt, torch_dequant_fp32, w4a16_inputs


def check(dx, dy, q, s, z, group):
    """Elementwise bounds from the two roundings.  Against the weight rounded to
    the activation type (as the kernels and the reference module hold it): the last rounding, u |dx|, and the fp32 accumulation, at
    most one 2^-23 step per 16-wide multiply-add of the N / 16 in the chain, of
    S = sum |dy| |w|.  Against the weight in full: u S more, from the rounding
    of the weight."""
    u = torch.finfo(dy.dtype).eps / 2
    w = torch_dequant_fp32(q, s, z, group).double()
    K = w.shape[0]
    wr = (((w / s.double().repeat_interleave(group, 0)).round()) * s.double().repeat_interleave(group, 0)).to(dy.dtype).double()
    d = dy.double()
    S = d.abs() @ w.abs().t()
    acc = 2.0 ** -23 * (dy.shape[1] / 16 + 8) * S
    tiny = 2.0 ** -25 if dy.dtype == torch.float16 else 0.0
    assert dx.shape == (dy.shape[0], K) and dx.dtype == dy.dtype
    ref = d @ wr.t()
    assert ((dx.double() - ref).abs() <= u * (ref.abs() + acc) + acc + tiny).all()
    full = d @ w.t()
    assert ((dx.double() - full).abs() <= u * (full.abs() + 2 * S) + acc + tiny).all()


def grads_in(M, K, N, group, dtype, seed=0):
    _, q, s, z = w4a16_inputs(1, K, N, group, dtype, seed=seed, device="cuda")
    g = torch.Generator().manual_seed(seed + 1)
    return (torch.randn(M, N, generator=g) * 0.1).to(tdt(dtype)).cuda(), q, s, z


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,K,N,group", [
    (1, 128, 32, 128), (2, 256, 1056, 256), (7, 96, 160, 32), (16, 192, 2048, 64), (5, 1408, 2080, 64), (1, 4096, 4096, 128), (3, 32, 64, 32), (16, 14336, 4096, 128), (17, 96, 96, 32),
    (129, 192, 224, 64), (130, 512, 1408, 256), (255, 2048, 1408, 64), (300, 320, 160, 64), (1000, 2048, 1408, 64),
    (777, 288, 4096, 32), (17, 2048, 1408, 256), (40, 1056, 8192, 32), (2048, 4096, 512, 128), (2000, 4096, 544, 256)])
def test_against_float64(M, K, N, group, dtype):
    args = grads_in(M, K, N, group, dtype)
    check(ops.w4a16_dgrad(*args, group), *args, group)
    assert ops.device_status() == 0


@pytest.mark.gpu
def test_one_weight_at_a_time():
    """Unit rows of dy give the dequantised weight's columns bit for bit."""
    _, q, s, z = grads_in(1, 256, 96, 32, "fp16", seed=4)
    eye = torch.eye(96, dtype=torch.float16, device="cuda")
    w = torch_dequant_fp32(q, s, z, 32).half()  # (nib - z) s: one rounding
    assert torch.equal(ops.w4a16_dgrad(eye, q, s, z, 32), w.t())
    assert torch.equal(torch.cat([ops.w4a16_dgrad(e, q, s, z, 32) for e in eye.split(16)]), w.t())


@pytest.mark.gpu
@pytest.mark.parametrize("M", [9, 40])
def test_small_and_large_gradients_in_fp16(M):
    """Rows of dy from the subnormals to near the type's end, and infinities and
    NaN that stay in their rows."""
    dy, q, s, z = grads_in(M, 256, 512, 64, "fp16", seed=6)
    dy = (dy.float() * torch.logspace(-5, 3, M, base=10.0, device="cuda")[:, None]).half()
    clean = ops.w4a16_dgrad(dy, q, s, z, 64)
    check(clean, dy, q, s, z, 64)
    dy[2, 7], dy[4, 9] = float("inf"), float("nan")
    dx = ops.w4a16_dgrad(dy, q, s, z, 64)
    rest = [m for m in range(M) if m not in (2, 4)]
    assert torch.equal(dx[rest], clean[rest])
    assert torch.isnan(dx[4]).all() and not torch.isfinite(dx[2]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 200])
def test_autograd_through_the_projection(M):
    x, q, s, z = w4a16_inputs(M, 512, 256, 128, "bf16", seed=7, device="cuda")
    x.requires_grad_()
    y = ops.w4a16_gemm(x, q, s, z, 128)
    dy = torch.randn_like(y)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert torch.equal(dx, ops.w4a16_dgrad(dy, q, s, z, 128))
    # the gradient of a scalar against differences of the module's linear map
    # (exact for a linear function up to the projection's own roundings)
    w = torch_dequant_fp32(q, s, z, 128).double()
    full = dy.double() @ w.t()
    u = 2.0 ** -8
    S = dy.double().abs() @ w.abs().t()
    assert ((dx.double() - full).abs() <= u * full.abs() + 2 * u * S + 1e-5 * S).all()
    # an expanded, non-contiguous gradient
    (d1,) = torch.autograd.grad(ops.w4a16_gemm(x, q, s, z, 128).sum(), x)
    assert torch.equal(d1, ops.w4a16_dgrad(torch.ones_like(y), q, s, z, 128))


@pytest.mark.gpu
def test_strided_misaligned_and_empty():
    dy, q, s, z = grads_in(40, 256, 128, 64, "fp16", seed=2)
    want = ops.w4a16_dgrad(dy, q, s, z, 64)
    assert torch.equal(ops.w4a16_dgrad(dy.t().contiguous().t(), q, s, z, 64), want)
    odd = torch.zeros(40 * 128 + 1, dtype=torch.float16, device="cuda")[1:].view(40, 128)
    odd.copy_(dy)
    assert torch.equal(ops.w4a16_dgrad(odd, q, s, z, 64), want)
    assert torch.equal(ops.w4a16_dgrad(dy, q, s.float(), z.float(), 64), want)
    assert ops.w4a16_dgrad(dy[:0], q, s, z, 64).shape == (0, 256)


@pytest.mark.gpu
def test_captured_on_two_streams():
    """Two graphs over the same weight, replayed at the same time on two streams."""
    dy, q, s, z = grads_in(16, 2048, 1024, 128, "bf16", seed=3)
    want = ops.w4a16_dgrad(dy, q, s, z, 128)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.w4a16_dgrad(dy, q, s, z, 128)
        graphs.append((g, out, torch.cuda.Stream()))
    for _ in range(5):
        for g, out, st in graphs:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                out.zero_()
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out, _ in graphs)


def test_refusals_without_gpu():
    dy, q = torch.zeros(4, 32, dtype=torch.float16), torch.zeros(128, 4, dtype=torch.int32)
    s = torch.zeros(1, 32, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.w4a16_dgrad(dy, q, s, s, 128)
    import kernelbench_harbor_b200 as pkg
    pkg.build()
    L, p = _lib.lib(), 16

    def call(M=16, N=4096, K=14336, group=128, dtype=0, dy=p, dx=p, ws=256):
        return L.b200q_w4a16_dgrad(dy, p, p, p, dx, M, N, K, group, dtype, p, ws, None)

    assert call(group=100) == call(dtype=2) == _lib.ERR_UNSUPPORTED
    assert call(N=4100) == call(dx=8) == _lib.ERR_ALIGN
    assert call(K=200) == call(M=-1) == call(dy=None) == call(M=1 << 24) == _lib.ERR_SHAPE
    assert call(ws=64) == _lib.ERR_WORKSPACE
    assert call(M=0) == _lib.OK


@pytest.mark.gpu
def test_refusals():
    dy, q, s, z = grads_in(4, 128, 32, 128, "fp16")
    for args, err in [((dy[:, :16], q, s, z, 128), ValueError), ((dy, q.long(), s, z, 128), TypeError),
                      ((dy, q, s, z, 100), ValueError), ((dy, q, s[:, :8], z, 128), ValueError),
                      ((dy.float(), q, s, z, 128), TypeError), ((dy[0], q, s, z, 128), ValueError)]:
        with pytest.raises(err):
            ops.w4a16_dgrad(*args)
    x = torch.zeros(4, 128, dtype=torch.float16, device="cuda", requires_grad=True)
    # scales that ask for a gradient run forward, as before, and have none
    y = ops.w4a16_gemm(x, q, s.clone().requires_grad_(), z, 128)
    with pytest.raises(RuntimeError, match="frozen"):
        y.sum().backward()


@pytest.mark.gpu
def test_from_a_thread_that_has_not_used_the_gpu():
    """A thread's first call (autograd's own thread makes one, too) once every
    attribute that a first call looks up is known."""
    import threading

    dy, q, s, z = grads_in(40, 256, 128, 64, "fp16", seed=3)
    x = torch.randn(40, 256, dtype=torch.float16, device="cuda")
    calls = [lambda: ops.w4a16_dgrad(dy, q, s, z, 64), lambda: ops.w4a16_dgrad(dy[:8], q, s, z, 64),
             lambda: ops.w4a16_gemm(x, q, s, z, 64)]
    for call in calls:
        want = call()
        torch.cuda.synchronize()
        got = []
        th = threading.Thread(target=lambda: got.append(call()))
        th.start()
        th.join()
        torch.cuda.synchronize()
        assert got and torch.equal(got[0], want)
