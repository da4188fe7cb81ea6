"""Load-balance loss, per-expert counts and the gradient of the logits,
against the definition in float64."""
import pytest
import torch

from kernelbench_harbor_b200 import _lib, ops

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def definition(logits, topi, mask, dloss=1.0):
    """(loss, counts, dlogits, scale): the definition in float64; scale is the
    sum of the magnitudes that dlogits' difference is taken of."""
    lg = logits.double()
    T, E = lg.shape
    live = ~torch.isneginf(lg).all(dim=1)
    if mask is not None:
        live &= mask
    n, k = int(live.sum()), topi.shape[1]
    counts = torch.zeros(E, dtype=torch.int64, device=lg.device)
    picked = topi[live].reshape(-1).long()
    picked = picked[(picked >= 0) & (picked < E)]
    counts += torch.bincount(picked, minlength=E)
    d, scale = torch.zeros_like(lg), torch.zeros_like(lg)
    if n == 0:
        return torch.zeros((), dtype=torch.float64, device=lg.device), counts, d, scale
    p = torch.softmax(lg[live], dim=1)
    f = counts.double() / (k * n)
    loss = E * (f * p.mean(dim=0)).sum()
    dot = p @ f
    d[live] = dloss * E / n * p * (f - dot[:, None])
    scale[live] = abs(dloss) * E / n * p * (f + dot[:, None])
    return loss, counts, d, scale


def bounds(logits, mask):
    """Relative error of a softmax probability and of the sums in fp32.  p: the
    rounding of v - max (|v - max| 2^-24 in the exponent), expf (2 ulp), the
    row's sum (8 in a lane and 5 shuffles), the reciprocal and the product.
    Sums over the rows: a lane's chain of T / 8 additions at most (one block of 8
    warps, one row each) plus the 5 + 8 + 32 of the joins."""
    lg = logits.double()[mask] if mask is not None else logits.double()
    lg = torch.where(torch.isneginf(lg), torch.nan, lg)
    finite = lg[~torch.isnan(lg)]
    spread = float(finite.max() - finite.min()) if finite.numel() else 0.0
    p = (spread + 2 * 2 + 13 + 2 + 2) * 2.0 ** -24
    return p, p + (logits.shape[0] / 8 + 45 + 8) * 2.0 ** -24


def check(logits, topi, mask, dloss=None):
    lg = logits.detach().requires_grad_()
    g = torch.tensor(1.0 if dloss is None else dloss, device="cuda")
    loss, counts = ops.moe_balance_loss(lg, topi, mask)
    (d,) = torch.autograd.grad(loss, lg, g)
    want, wcounts, wd, scale = definition(logits, topi, mask, float(g))
    ep, es = bounds(logits, mask)
    assert loss.dtype == torch.float32 and loss.dim() == 0 and counts.dtype == torch.int32
    assert torch.equal(counts.long(), wcounts)
    assert abs(loss.double() - want) <= es * want
    u = torch.finfo(logits.dtype).eps / 2
    tiny = 2.0 ** -25 if logits.dtype == torch.float16 else 2.0 ** -134  # half a subnormal step
    # the dot product adds 8 + 5 roundings, the factors 6 more; the last rounding is u
    tol = (2 * ep + 20 * 2.0 ** -24) * scale + u * wd.abs() + tiny
    assert d.dtype == logits.dtype
    bad = (d.double() - wd).abs() > tol * (1 + u)
    assert not bad.any(), (d.double() - wd).abs()[bad].max()
    # without a gradient: the same bits
    loss2, counts2 = ops.moe_balance_loss(logits, topi, mask)
    assert torch.equal(loss2, loss.detach()) and torch.equal(counts2, counts)
    return loss, counts, d


def inputs(T, E, k, dtype, seed=0, masked=0.0):
    g = torch.Generator().manual_seed(seed + 1000 * E + T)
    logits = (torch.randn(T, E, generator=g) * 2 + torch.randn(E, generator=g)).to(DTYPES[dtype])
    topi = torch.topk(logits.float(), k, dim=1).indices.to(torch.int32)
    mask = torch.rand(T, generator=g) >= masked if masked else None
    return logits.cuda(), topi.cuda(), mask.cuda() if mask is not None else None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("T,E,k,masked", [
    (1, 2, 1, 0.0), (1, 8, 2, 0.0), (7, 3, 2, 0.0), (512, 8, 2, 0.25), (333, 17, 4, 0.5), (100, 60, 2, 0.0),
    (2049, 64, 8, 0.1), (257, 100, 6, 0.0), (1000, 256, 8, 0.3), (33, 255, 1, 0.0), (20000, 16, 2, 0.2)])
def test_against_definition(T, E, k, masked, dtype):
    logits, topi, mask = inputs(T, E, k, dtype, masked=masked)
    # a loss weight times a loss scale, so that fp16 gradients are in range
    check(logits, topi, mask, dloss=0.01 * 2.0 ** 14)


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the float64 loss with the counts held (h^2 error
    of a loss whose third derivative is below E, at h = 1e-4)."""
    logits, topi, _ = inputs(5, 6, 2, "fp32")
    _, counts, d = check(logits, topi, None)
    f = counts.double() / 10
    loss = lambda lg: 6 * (f * torch.softmax(lg, dim=1).mean(dim=0)).sum()  # noqa: E731
    lg, h = logits.double(), 1e-4
    for t in range(5):
        for e in range(6):
            up, down = lg.clone(), lg.clone()
            up[t, e] += h
            down[t, e] -= h
            num = (loss(up) - loss(down)) / (2 * h)
            assert abs(num - d[t, e].double()) <= 6 * h * h + 1e-15 / h + 1e-6 * 6 / 5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_masked_and_empty_rows(dtype):
    logits, topi, _ = inputs(64, 8, 2, dtype, seed=3)
    logits[5] = float("-inf")            # no expert at all: not live
    logits[6, 2:] = float("-inf")        # two experts left
    logits[7], logits[8] = float("nan"), float("inf")
    mask = torch.ones(64, dtype=torch.bool, device="cuda")
    mask[7], mask[8] = False, False      # NaN and inf in padding stay there
    topi[9] = -1                         # both choices dropped
    _, _, d = check(logits, topi, mask)
    assert (d[5] == 0).all() and (d[7:9] == 0).all()
    none = torch.zeros(64, dtype=torch.bool, device="cuda")
    loss, counts, d = check(logits, topi, none)
    assert loss.item() == 0 and counts.sum() == 0 and (d == 0).all()
    # a NaN in a live row is not hidden
    assert torch.isnan(ops.moe_balance_loss(logits, topi)[0])


@pytest.mark.gpu
def test_no_tokens():
    lg = torch.empty(0, 8, device="cuda", requires_grad=True)
    loss, counts = ops.moe_balance_loss(lg, torch.empty(0, 2, dtype=torch.int32, device="cuda"))
    (d,) = torch.autograd.grad(loss, lg)
    assert loss.item() == 0 and counts.tolist() == [0] * 8 and d.shape == (0, 8)


@pytest.mark.gpu
def test_index_out_of_range_sets_the_status():
    logits, topi, _ = inputs(40, 8, 2, "fp32", seed=5)
    ops.moe_balance_loss(logits, topi)
    assert ops.device_status() == 0
    topi[3, 1] = 8
    check(logits, topi, None)
    assert ops.device_status() & 2
    assert ops.device_status() == 0
    wide = topi.long()
    wide[4, 0] = 2 ** 32 + 1  # not expert 1
    wide[5, 1] = -2 ** 40
    _, counts = ops.moe_balance_loss(logits, wide)
    assert torch.equal(counts.long(), definition(logits, wide, None)[1])
    assert ops.device_status() & 2


@pytest.mark.gpu
def test_gradient_twice_and_once_differentiable():
    """A retained graph gives the same gradient again; the gradient itself has none."""
    logits, topi, mask = inputs(50, 8, 2, "fp32", seed=21, masked=0.2)
    lg = logits.requires_grad_()
    loss, _ = ops.moe_balance_loss(lg, topi, mask)
    (d1,) = torch.autograd.grad(loss, lg, retain_graph=True)
    (d2,) = torch.autograd.grad(3 * loss, lg, create_graph=True)
    torch.testing.assert_close(d2, 3 * d1, rtol=2 ** -22, atol=0)
    with pytest.raises(RuntimeError):
        d2.square().sum().backward()


@pytest.mark.gpu
def test_layouts_streams_and_repeat():
    """Strided logits, int64 indices, a stream of their own, misaligned rows;
    the same bits every time."""
    logits, topi, mask = inputs(5000, 32, 2, "bf16", seed=9, masked=0.2)
    loss, counts, d = check(logits, topi, mask)
    wide = torch.zeros(5000, 64, dtype=torch.bfloat16, device="cuda")
    wide[:, 32:] = logits
    odd = torch.zeros(5000 * 32 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(5000, 32)
    odd.copy_(logits)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for lg in (wide[:, 32:], odd):
            l2, c2, d2 = check(lg, topi.long(), mask)
            assert torch.equal(l2, loss) and torch.equal(c2, counts) and torch.equal(d2, d)
    s.synchronize()


@pytest.mark.gpu
def test_captured_and_replayed_with_the_route():
    """moe_route and the loss with its gradient in one graph, replayed on new logits."""
    logits, _, mask = inputs(3000, 8, 2, "bf16", seed=11, masked=0.1)
    static = logits.clone().requires_grad_()

    def step():
        topi = ops.moe_route(static.detach())[0]
        loss, counts = ops.moe_balance_loss(static, topi, mask)
        return loss, counts, torch.autograd.grad(loss, static)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (12, 13):
        new = inputs(3000, 8, 2, "bf16", seed=seed)[0]
        with torch.no_grad():
            static.copy_(new)
        graph.replay()
        want = check(new, ops.moe_route(new)[0], mask)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals_on_cpu():
    lg, topi = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.moe_balance_loss(lg, topi)


@pytest.mark.gpu
def test_refusals():
    lg, topi = torch.zeros(4, 8, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    mask = torch.ones(4, dtype=torch.bool, device="cuda")
    for args, err in [((lg, topi[:3]), ValueError), ((lg[0], topi), ValueError), ((lg.double(), topi), TypeError),
                      ((lg, topi.float()), TypeError), ((lg, topi, mask.int()), ValueError),
                      ((lg, topi, mask[:3]), ValueError), ((lg, topi.cpu()), ValueError),
                      ((lg[:, :1], topi), _lib.B200QError), ((lg.repeat(1, 33), topi), _lib.B200QError),
                      ((lg, topi.repeat(1, 5)), _lib.B200QError), ((lg, topi[:, :0]), _lib.B200QError)]:
        with pytest.raises(err):
            ops.moe_balance_loss(*args)


def test_c_entry_refuses_before_the_gpu():
    import kernelbench_harbor_b200 as pkg
    pkg.build()
    L, p = _lib.lib(), 16

    def call(T=4, E=8, k=2, dtype=2, logits=p, scratch=1 << 20):
        return L.b200q_moe_balance(logits, p, None, T, E, k, dtype, p, p, p, p, scratch, None, None)

    assert call(E=1) == call(E=257) == call(k=0) == call(k=9) == call(T=-1) == _lib.ERR_SHAPE
    assert call(E=3, k=4) == call(logits=None) == call(T=(1 << 27) + 1) == _lib.ERR_SHAPE
    assert call(dtype=3) == _lib.ERR_UNSUPPORTED
    assert call(scratch=4) == _lib.ERR_WORKSPACE
    assert L.b200q_moe_balance_grad(None, None, p, p, 4, 8, 2, p, None) == _lib.ERR_SHAPE
    assert L.b200q_moe_balance_grad(p, None, p, p, 4, 8, 5, p, None) == _lib.ERR_UNSUPPORTED
    assert L.b200q_moe_balance_grad(p, None, p, p, 0, 8, 2, p, None) == _lib.OK
