"""Adapters of many requests beside one shared projection: lora_plan,
lora_apply and its gradients, and the W4A16 module that uses them, against
float64."""
import pytest
import torch

from kernelbench_harbor_b200 import _lib, ops
from tests.helpers import tdt, torch_dequant_fp32, w4a16_inputs

STEP = 2.0 ** -23  # one fp32 accumulation step of a multiply-add chain


def ids_of(T, L, kind, seed=0):
    g = torch.Generator().manual_seed(seed + T)
    if kind == "runs":  # requests one after another, some without an adapter
        out = []
        while len(out) < T:
            out += [int(torch.randint(-1, L, (1,), generator=g))] * int(torch.randint(1, 40, (1,), generator=g))
        return torch.tensor(out[:T], dtype=torch.int64)
    if kind == "mixed":
        return torch.randint(-1, L, (T,), generator=g)
    if kind == "one":
        return torch.full((T,), L - 1)
    return torch.full((T,), -1)


def inputs(T, D, N, r, L, dtype, kind, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * T + D + r)
    dt = tdt(dtype)
    n = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dt).cuda()  # noqa: E731
    return dict(base=n(T, N), x=n(T, D), A=n(L, D, r, std=D ** -0.5), B=n(L, r, N, std=r ** -0.5),
                dy=n(T, N, std=0.3), ids=ids_of(T, L, kind, seed).cuda(),
                scaling=(torch.rand(L, generator=g) * 1.5 + 0.5).cuda())


def pair(x, P, Q, s, ids, base=None):
    """(mid, out, mid's error bound, out's error bound before its last rounding)
    of mid = s x . P[id], out = base + mid . Q[id], float64.  The bounds: a chain
    of K / 16 multiply-adds of 16 and 40 joins, one step each of the sum of
    magnitudes; the split of mid into two halves of the type (u^2 of a value,
    and 2^-24 of the row's largest at most); r / 16 + 4 steps of the second chain."""
    x, P, Q = x.double(), P.double(), Q.double()
    T, N = x.shape[0], Q.shape[2]
    r = P.shape[2]
    mid, emid = (torch.zeros(T, r, dtype=torch.float64, device=x.device) for _ in range(2))
    out = base.double().clone() if base is not None else torch.zeros(T, N, dtype=torch.float64, device=x.device)
    eout = torch.zeros_like(out)
    for a in range(P.shape[0]):
        t = torch.nonzero(ids == a).flatten()
        if not len(t):
            continue
        sa = 1.0 if s is None else s[a].double()
        m = sa * (x[t] @ P[a])
        mag = sa * (x[t].abs() @ P[a].abs())
        mid[t], emid[t] = m, (x.shape[1] / 16 + 40) * STEP * mag
        e = emid[t] + 2.0 ** -16 * m.abs() + 2.0 ** -24 * m.abs().amax(dim=1, keepdim=True)
        out[t] += m @ Q[a]
        eout[t] = e @ Q[a].abs() + (r / 16 + 4) * STEP * (m.abs() @ Q[a].abs()) + STEP * out[t].abs()
    return mid, out, emid, eout


def close(got, want, err, u_dtype):
    u = torch.finfo(u_dtype).eps / 2
    tiny = 2.0 ** -25 if u_dtype == torch.float16 else 0.0
    bad = (got.double() - want).abs() > err + u * (want.abs() + err) + tiny
    # a value of at least the largest finite one plus half a step (fp16: 65504 + 16,
    # the step below 65536 being 32) rounds to infinity of its sign
    top = torch.finfo(u_dtype).max * (1 + u / (2 - 2 * u))
    bad &= ~(torch.isinf(got) & (want.abs() + err >= top) & (torch.sign(got) == torch.sign(want)))
    assert got.dtype == u_dtype and got.shape == want.shape
    assert not bad.any(), ((got.double() - want).abs()[bad].max(), int(bad.sum()))


def grads(wide, thin, ethin, ids, L):
    """(sum_t wide^T thin, its bound) per adapter: [L, W, r]."""
    wide = wide.double()
    out = torch.zeros(L, wide.shape[1], thin.shape[1], dtype=torch.float64, device=wide.device)
    err = torch.zeros_like(out)
    for a in range(L):
        t = torch.nonzero(ids == a).flatten()
        if not len(t):
            continue
        w, m = wide[t], thin[t]
        e = ethin[t] + 2.0 ** -16 * m.abs() + 2.0 ** -24 * m.abs().max()
        out[a] = w.t() @ m
        err[a] = w.abs().t() @ e + (len(t) / 16 + 48) * STEP * (w.abs().t() @ m.abs())
    return out, err


def check(c, train=True, plan=None):
    dt = c["x"].dtype
    L = c["A"].shape[0]
    plan = plan if plan is not None else ops.lora_plan(c["ids"], L)
    leaves = [c[k].detach().clone().requires_grad_(train) for k in ("base", "x", "A", "B")]
    y = ops.lora_apply(*leaves, plan, c["scaling"])
    lo, want, elo, ey = pair(c["x"], c["A"], c["B"], c["scaling"], c["ids"], c["base"])
    close(y.detach(), want, ey, dt)
    none = (c["ids"] < 0) | (c["ids"] >= L)
    assert torch.equal(y.detach()[none], c["base"][none])
    if not train:
        return y, None
    dbase, dx, dA, dB = torch.autograd.grad(y, leaves, c["dy"])
    At, Bt = c["A"].transpose(1, 2), c["B"].transpose(1, 2)
    dlo, wdx, edlo, edx = pair(c["dy"], Bt, At, c["scaling"], c["ids"])
    close(dx, wdx, edx, dt)
    close(dA, *grads(c["x"], dlo, edlo, c["ids"], L), dt)
    wB, eB = grads(c["dy"], lo, elo, c["ids"], L)
    close(dB, wB.transpose(1, 2), eB.transpose(1, 2), dt)
    assert torch.equal(dbase, c["dy"]) and (dx[none] == 0).all()
    return y.detach(), (dx, dA, dB)


# ---------------------------------------------------------------- plan
@pytest.mark.gpu
@pytest.mark.parametrize("T,L,kind", [(1, 1, "one"), (1, 5, "none"), (31, 3, "mixed"), (64, 64, "mixed"),
                                      (1000, 7, "runs"), (5000, 1023, "mixed"), (70000, 4, "runs"), (4097, 2, "one")])
def test_plan(T, L, kind):
    ids = ids_of(T, L, kind)
    words = ops.lora_plan(ids.cuda(), L).data.cpu()
    up4 = lambda v: (v + 3) // 4 * 4  # noqa: E731
    seg = torch.where(ids < 0, torch.full_like(ids, L), ids)
    off = torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(seg, minlength=L + 1).cumsum(0)])
    assert torch.equal(words[8:8 + L + 2].long(), off)
    at = up4(8 + L + 2)
    order = words[at:at + T].long()
    assert torch.equal(order, torch.sort(seg, stable=True).indices)
    at = up4(at + T)
    for rows, count in ((16, int(words[0])), (128, int(words[1]))):
        want = [(a if a < L else -1, s, min(rows, int(off[a + 1]) - s)) for a in range(L + 1)
                for s in range(int(off[a]), int(off[a + 1]), rows)]
        got = words[at:at + 4 * count].view(-1, 4)[:, :3].tolist()
        assert [tuple(g) for g in got] == want
        at += 4 * min(T, T // rows + L + 1)


@pytest.mark.gpu
def test_ids_out_of_range_count_as_none():
    c = inputs(40, 64, 64, 8, 3, "bf16", "mixed")
    check(c)
    assert ops.device_status() == 0
    c["ids"][5], c["ids"][6], c["ids"][7] = 3, -2, 2 ** 40
    check(c)
    assert ops.device_status() & 2
    assert ops.device_status() == 0


# ---------------------------------------------------------------- values and gradients
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("T,D,N,r,L,kind", [
    (1, 64, 64, 8, 1, "one"), (5, 8, 8, 8, 2, "mixed"), (260, 8, 16, 8, 2, "runs"), (1, 4096, 4096, 16, 8, "one"), (1, 128, 256, 64, 2, "none"), (3, 32, 8, 1, 2, "mixed"),
    (16, 264, 40, 16, 1, "one"), (17, 4096, 1408, 16, 2, "one"), (64, 512, 768, 32, 64, "mixed"),
    (64, 4096, 4096, 16, 8, "mixed"), (100, 257, 129, 33, 3, "mixed"), (129, 1000, 264, 64, 2, "runs"),
    (256, 2048, 512, 24, 5, "runs"), (257, 128, 128, 16, 3, "runs"), (300, 4100, 64, 12, 2, "mixed"),
    (300, 70, 333, 5, 4, "runs"), (700, 1408, 2048, 8, 60, "runs"), (1000, 512, 1152, 64, 1, "one"),
    (1300, 72, 2056, 48, 3, "runs"), (2049, 3584, 256, 32, 5, "mixed"), (600, 264, 264, 16, 2, "none"),
    (1100, 1096, 1096, 36, 2, "mixed"), (4100, 264, 264, 60, 3, "runs"), (1024, 1024, 1032, 64, 1, "none")])
def test_against_float64(T, D, N, r, L, kind, dtype):
    check(inputs(T, D, N, r, L, dtype, kind))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 400])
def test_gradient_against_differences(T):
    """The operator is linear in x, in A and in B: f(v + e) - f(v) of its float64
    form is the gradient's product with e, up to the gradient's own rounding."""
    c = inputs(T, 96, 64, 8, 2, "bf16", "runs")
    _, (dx, dA, dB) = check(c)
    u = 2.0 ** -8
    for name, d in (("x", dx), ("A", dA), ("B", dB)):
        e = torch.randn_like(c[name])
        moved = {**{k: c[k].double() for k in ("x", "A", "B")}}
        moved[name] = moved[name] + e.double()
        f = lambda v: (pair(v["x"], v["A"], v["B"], c["scaling"], c["ids"])[1] * c["dy"].double()).sum()  # noqa: E731
        num = f(moved) - f({k: c[k].double() for k in ("x", "A", "B")})
        terms = (d.double() * e.double()).abs().sum()
        assert abs(num - (d.double() * e.double()).sum()) <= 2 * u * terms


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("T", [48, 512])
def test_row_between_keeps_fp32(T, dtype):
    """With B the identity and base minus the rounded row, y is the part of lo
    that its type would have dropped."""
    c = inputs(T, 256, 16, 16, 1, dtype, "one")
    c["B"] = torch.eye(16, dtype=c["x"].dtype, device="cuda")[None]
    lo, _, elo, _ = pair(c["x"], c["A"], c["B"], c["scaling"], c["ids"])
    c["base"] = -lo.to(c["x"].dtype)
    y = ops.lora_apply(c["base"], c["x"], c["A"], c["B"], c["ids"], c["scaling"])
    close(y, lo + c["base"].double(), elo + 2.0 ** -16 * lo.abs() + 2.0 ** -24 * lo.abs().amax(dim=1, keepdim=True),
          c["x"].dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [33, 700])
def test_fp16_rows_outside_the_types_range(T):
    """lo above 65504 and below the smallest fp16, with results inside it: rows
    of very different sizes side by side, in the products and in the sums over tokens."""
    c = inputs(T, 128, 64, 16, 2, "fp16", "mixed")
    size = torch.logspace(-3, 3, T, base=10.0)[torch.randperm(T, generator=torch.Generator().manual_seed(1))].cuda()
    c["x"] = (c["x"].float() * size[:, None]).half()
    c["A"] = (c["A"].float() * 100).half()       # lo from ~1e-1 to ~1e5
    c["B"] = (c["B"].float() * 1e-3).half()
    assert pair(c["x"], c["A"], c["B"], c["scaling"], c["ids"])[0].abs().max() > 65504
    check(c)
    c["A"], c["dy"] = (c["A"].float() * 1e-7).half(), (c["dy"].float() * 1e-3).half()  # lo from ~1e-8
    check(c)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [30, 400])
def test_nonfinite_rows_stay_alone(T):
    c = inputs(T, 64, 72, 8, 2, "bf16", "mixed")
    c["ids"][3], c["ids"][4], c["ids"][5] = 0, -1, 1
    clean = ops.lora_apply(c["base"], c["x"], c["A"], c["B"], c["ids"], c["scaling"])
    c["x"][3], c["x"][4] = float("inf"), float("nan")
    y = ops.lora_apply(c["base"], c["x"], c["A"], c["B"], c["ids"], c["scaling"])
    others = [t for t in range(T) if t != 3]
    assert torch.equal(y[others], clean[others])  # a row without an adapter never reads x
    assert not torch.isfinite(y[3]).any()
    # one infinite value of x: lo is +-inf where A is not 0, y is +-inf or NaN, as float64 has it
    c["x"][3] = 0
    c["x"][3, 0] = float("inf")
    c["A"][0, 0], c["B"][0] = 1.0, c["B"][0].abs() + 0.5
    y = ops.lora_apply(c["base"], c["x"], c["A"], c["B"], c["ids"], c["scaling"])
    assert (y[3] == float("inf")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [50, 500])
def test_masked_rows_of_the_output_gradient(T):
    """Padding tokens: a zero gradient row gives zeros and leaves the sums alone."""
    c = inputs(T, 128, 96, 8, 2, "bf16", "runs")
    c["dy"][T // 2:] = 0
    _, (dx, dA, dB) = check(c)
    assert (dx[T // 2:] == 0).all()


# ---------------------------------------------------------------- calls
@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 600])
def test_layouts_and_types(T):
    c = inputs(T, 256, 128, 16, 3, "bf16", "runs")
    plan = ops.lora_plan(c["ids"], 3)
    want = ops.lora_apply(c["base"], c["x"], c["A"], c["B"], plan, c["scaling"])
    apply = lambda **kw: ops.lora_apply(*[{**c, **kw}[k] for k in ("base", "x", "A", "B")], plan, c["scaling"])  # noqa: E731
    wide = torch.zeros(T, 512, dtype=torch.bfloat16, device="cuda")
    wide[:, 128:384] = c["x"]
    odd = torch.zeros(T * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(T, 256)
    odd.copy_(c["x"])
    assert torch.equal(apply(x=wide[:, 128:384]), want) and torch.equal(apply(x=odd), want)
    assert torch.equal(apply(A=c["A"].transpose(1, 2).contiguous().transpose(1, 2)), want)
    assert torch.equal(apply(A=c["A"].float(), B=c["B"].float()), want)
    assert torch.equal(ops.lora_apply(c["base"], c["x"], c["A"], c["B"], c["ids"].int(), c["scaling"]), want)
    out = torch.empty_like(want)
    assert ops.lora_apply(c["base"], c["x"], c["A"], c["B"], plan, c["scaling"], out=out) is out
    assert torch.equal(out, want)
    base = c["base"].clone()
    assert ops.lora_apply(base, c["x"], c["A"], c["B"], plan, c["scaling"], out=base) is base
    assert torch.equal(base, want)
    one = ops.lora_apply(c["base"], c["x"], c["A"], c["B"], plan)
    assert torch.equal(one, ops.lora_apply(c["base"], c["x"], c["A"], c["B"], plan, torch.ones(3, device="cuda")))
    # fp32 master adapters get fp32 gradients
    A32 = c["A"].float().requires_grad_()
    (g,) = torch.autograd.grad(apply(A=A32), A32, c["dy"])
    assert g.dtype == torch.float32
    # an expanded gradient
    A = c["A"].clone().requires_grad_()
    (g1,) = torch.autograd.grad(apply(A=A).sum(), A)
    (g2,) = torch.autograd.grad(apply(A=A), A, torch.ones_like(want))
    assert torch.equal(g1, g2)


@pytest.mark.gpu
def test_gradients_one_at_a_time():
    c = inputs(300, 64, 128, 8, 2, "fp16", "runs")
    _, (dx, dA, dB) = check(c)
    for name, want in (("x", dx), ("A", dA), ("B", dB), ("base", c["dy"])):
        leaf = c[name].clone().requires_grad_()
        kw = {**c, name: leaf}
        (g,) = torch.autograd.grad(ops.lora_apply(kw["base"], kw["x"], kw["A"], kw["B"], c["ids"], c["scaling"]), leaf, c["dy"])
        assert torch.equal(g, want)


@pytest.mark.gpu
def test_once_differentiable():
    c = inputs(40, 64, 64, 8, 2, "bf16", "runs")
    A = c["A"].float().requires_grad_()
    y = ops.lora_apply(c["base"], c["x"], A, c["B"], c["ids"], c["scaling"])
    (g,) = torch.autograd.grad(y.float().square().sum(), A, create_graph=True)
    with pytest.raises(RuntimeError):
        g.square().sum().backward()


@pytest.mark.gpu
def test_no_tokens():
    A, B = (torch.randn(2, 64, 8, device="cuda").half().requires_grad_(), torch.randn(2, 8, 32, device="cuda").half().requires_grad_())
    x, base = torch.zeros(0, 64, dtype=torch.float16, device="cuda"), torch.zeros(0, 32, dtype=torch.float16, device="cuda")
    ids = torch.zeros(0, dtype=torch.int64, device="cuda")
    y = ops.lora_apply(base, x, A, B, ids)
    dA, dB = torch.autograd.grad(y, (A, B), y.detach())
    assert y.shape == (0, 32) and (dA == 0).all() and (dB == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,N,r", [(64, 512, 384, 16), (1000, 512, 384, 16), (1200, 1024, 1096, 64)])
def test_the_same_bits_on_other_streams_and_in_graphs(T, D, N, r):
    """Forward and backward captured twice, replayed at the same time on two
    streams, on new inputs."""
    c = inputs(T, D, N, r, 4, "bf16", "runs")
    leaves = [c[k].clone().requires_grad_() for k in ("x", "A", "B")]
    plan = ops.lora_plan(c["ids"], 4)

    def step():
        y = ops.lora_apply(c["base"], *leaves, plan, c["scaling"])
        return (y, *torch.autograd.grad(y, leaves, c["dy"]))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out, torch.cuda.Stream()))
    with torch.no_grad():
        leaves[0].mul_(-1.5)
        c["dy"].add_(0.25)
    want = step()
    for _ in range(3):
        for g, out, st in graphs:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for _, out, _ in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,r,L", [(40, 264, 16, 3), (700, 264, 32, 3), (700, 264, 32, 60), (1300, 1032, 60, 3), (1300, 1032, 60, 40)])
def test_in_place_on_the_base(T, N, r, L):
    """y over base, rows without an adapter left as they are; the same bits as beside it."""
    c = inputs(T, 264, N, r, L, "fp16", "mixed")
    plan = ops.lora_plan(c["ids"], L)
    args = (c["x"], c["A"], c["B"], plan, c["scaling"])
    want = ops.lora_apply(c["base"], *args)
    y = c["base"].clone()
    assert ops.lora_apply(y, *args, out=y) is y
    assert torch.equal(y, want) and torch.equal(y[c["ids"] < 0], c["base"][c["ids"] < 0])


# ---------------------------------------------------------------- the module
@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 300])
def test_module_forward_and_gradients(T):
    from kernelbench_harbor_b200.modules import LoRAW4A16Linear
    x, q, s, z = w4a16_inputs(T, 512, 256, 128, "bf16", seed=T, device="cuda")
    c = inputs(T, 512, 256, 16, 3, "bf16", "runs")
    layer = LoRAW4A16Linear()
    base = ops.w4a16_gemm(x, q, s, z, 128)
    want = ops.lora_apply(base, x, c["A"], c["B"], c["ids"], c["scaling"])
    with torch.no_grad():
        y = layer(x.view(1, T, 512), q, s, z, c["A"], c["B"], c["ids"].view(1, T), c["scaling"])
    assert torch.equal(y[0], want)
    leaves = [t.clone().requires_grad_() for t in (x, c["A"], c["B"])]
    y = layer(leaves[0], q, s, z, leaves[1], leaves[2], c["ids"], c["scaling"])
    assert torch.equal(y, want)
    dx, dA, dB = torch.autograd.grad(y, leaves, c["dy"])
    w = torch_dequant_fp32(q, s, z, 128).double()
    dy = c["dy"].double()
    dlo, part, edlo, edx = pair(c["dy"], c["B"].transpose(1, 2), c["A"].transpose(1, 2), c["scaling"], c["ids"])
    u = 2.0 ** -8
    # the frozen weight's bf16 rounding, the first summand's and the sum's
    S = dy.abs() @ w.abs().t()
    full = dy @ w.t()
    assert ((dx.double() - full - part).abs() <= edx + (u + 1e-5) * S + 2.1 * u * (full.abs() + part.abs())).all()
    close(dA, *grads(x, dlo, edlo, c["ids"], 3), torch.bfloat16)
    lo, _, elo, _ = pair(x, c["A"], c["B"], c["scaling"], c["ids"])
    wB, eB = grads(c["dy"], lo, elo, c["ids"], 3)
    close(dB, wB.transpose(1, 2), eB.transpose(1, 2), torch.bfloat16)
    # one gradient at a time, and the operator that the module calls
    for i, want in enumerate((dx, dA, dB)):
        one = [t.detach().requires_grad_(i == k) for k, t in enumerate(leaves)]
        y = ops.lora_w4a16(one[0], q, s, z, 128, one[1], one[2], c["ids"], c["scaling"])
        assert torch.equal(torch.autograd.grad(y, one[i], c["dy"])[0], want)
    with pytest.raises(RuntimeError, match="frozen"):
        ops.lora_w4a16(leaves[0], q, s.clone().requires_grad_(), z, 128, c["A"], c["B"], c["ids"]).sum().backward()
    for bad in ((x, q[:, :16], s, z, 128, c["A"], c["B"]), (x, q, s, z, 64, c["A"], c["B"]),
                (x[:, :256], q, s, z, 128, c["A"], c["B"]), (x.float(), q, s, z, 128, c["A"], c["B"])):
        with pytest.raises((ValueError, TypeError)):
            ops.lora_w4a16(*bad, c["ids"])


@pytest.mark.gpu
def test_adapters_and_router_fitted_together():
    """A training step as a user writes it: a router over 8 experts with the
    balance loss, two adapter projections one after the other, one backward
    pass; then the batch served in a captured decode step."""
    from kernelbench_harbor_b200.modules import LoRAW4A16Linear, MoEBalanceLoss
    T, D, H, r, L, E = 200, 256, 512, 8, 3, 8
    x, q1, s1, z1 = w4a16_inputs(T, D, H, 64, "bf16", seed=1, device="cuda")
    _, q2, s2, z2 = w4a16_inputs(1, H, D, 64, "bf16", seed=2, device="cuda")
    c1, c2 = inputs(T, D, H, r, L, "bf16", "runs"), inputs(T, H, D, r, L, "bf16", "runs")
    par = [t.requires_grad_() for t in (c1["A"], c1["B"], c2["A"], c2["B"])]
    router = (torch.randn(D, E, device="cuda") * 0.1).bfloat16().requires_grad_()
    layer, balance, plan = LoRAW4A16Linear(), MoEBalanceLoss(), ops.lora_plan(c1["ids"], L)
    mask = torch.arange(T, device="cuda") < T - 9

    def step():
        h = layer(x, q1, s1, z1, par[0], par[1], plan, c1["scaling"])
        h = h * 0.05
        y = layer(h, q2, s2, z2, par[2], par[3], plan, c1["scaling"])
        logits = x @ router
        topi = ops.moe_route(logits.detach())[0]
        aux, counts = balance(logits, topi, mask)
        loss = (y.float() * mask[:, None]).square().mean() + 0.01 * aux
        return loss, counts, torch.autograd.grad(loss, [*par, router]), topi

    loss, counts, g, topi = step()
    assert int(counts.sum()) == 2 * (T - 9) and torch.isfinite(loss)
    for t, d in zip([*par, router], g):
        assert d.shape == t.shape and torch.isfinite(d.float()).all() and (d != 0).any()
    again = step()
    assert torch.equal(again[0], loss) and all(torch.equal(a, b) for a, b in zip(again[2], g))
    # the router's gradient against float64
    p = torch.softmax((x @ router).detach().double(), dim=1)[mask]
    f = counts.double() / (2 * (T - 9))
    dl = 0.01 * E / (T - 9) * p * (f - (p @ f)[:, None])
    want = x[mask].double().t() @ dl
    tol = 3 * 2.0 ** -8 * (x[mask].double().abs().t() @ dl.abs()) + 2.0 ** -8 * want.abs()
    assert ((g[4].double() - want).abs() <= tol).all()
    # serving: the whole step in one graph, new tokens and new requests on replay
    ids, xs = c1["ids"][:64].clone(), x[:64].clone()

    def serve():
        plan = ops.lora_plan(ids, L)
        h = layer(xs, q1, s1, z1, par[0], par[1], plan, c1["scaling"]) * 0.05
        return layer(h, q2, s2, z2, par[2], par[3], plan, c1["scaling"])

    with torch.no_grad():
        serve()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = serve()
        ids.copy_(c1["ids"][64:128])
        xs.copy_(x[64:128])
        graph.replay()
        assert torch.equal(out, serve())


# ---------------------------------------------------------------- refusals
def test_refusals_without_gpu():
    z = torch.zeros
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.lora_plan(z(4, dtype=torch.int64), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.lora_apply(z(4, 8), z(4, 8), z(2, 8, 4), z(2, 4, 8), z(4, dtype=torch.int64))
    import kernelbench_harbor_b200 as pkg
    pkg.build()
    L, p = _lib.lib(), 16
    assert L.b200q_lora_plan_bytes(-1, 4) == L.b200q_lora_plan_bytes(4, 0) == L.b200q_lora_plan_bytes(4, 1024) == 0
    n = L.b200q_lora_plan_bytes(64, 8)
    assert n >= 4 * (8 + 10 + 64)
    assert L.b200q_lora_plan(p, 64, 8, p, n - 4, None, None) == _lib.ERR_WORKSPACE
    assert L.b200q_lora_plan(None, 64, 8, p, n, None, None) == _lib.ERR_SHAPE
    assert L.b200q_lora_plan(p, 64, 8, 20, n, None, None) == _lib.ERR_ALIGN
    assert L.b200q_lora_plan(p, 64, 0, p, n, None, None) == L.b200q_lora_plan(p, (1 << 24) + 1, 8, p, n, None, None) == _lib.ERR_SHAPE

    def call(T=64, D=64, N=64, r=8, nl=4, dtype=0, x=p, y=p, lo=p):
        return L.b200q_lora_apply(x, p, p, p, None, p, T, D, N, r, nl, dtype, y, lo, None, None)

    assert call(r=65) == call(r=0) == call(D=0) == call(N=1 << 23) == call(nl=1024) == call(T=-1) == _lib.ERR_SHAPE
    assert call(x=None) == call(lo=None, T=257) == call(y=None) == _lib.ERR_SHAPE
    assert call(y=24) == call(x=8) == _lib.ERR_ALIGN
    assert call(dtype=2) == _lib.ERR_UNSUPPORTED
    assert call(T=0) == _lib.OK

    need = L.b200q_lora_backward_scratch_bytes(64, 64, 64, 8, 4, 0)
    assert need >= L.b200q_lora_mid_bytes(64, 8) > 0
    assert L.b200q_lora_backward_scratch_bytes(64, 64, 64, 65, 4, 0) == 0

    def back(T=64, r=8, x=p, dy=p, A=p, dx=p, dA=p, dB=p, lo=p, scratch=p, nbytes=need):
        return L.b200q_lora_backward(x, dy, None, A, p, None, p, lo, T, 64, 64, r, 4, 0, scratch, nbytes, dx, dA, dB,
                                     None, None)

    assert back(x=None) == back(dy=None) == back(A=None) == back(lo=None) == back(r=65) == _lib.ERR_SHAPE
    assert back(scratch=None) == back(nbytes=need - 4) == _lib.ERR_WORKSPACE
    assert back(dB=8) == back(dx=4) == _lib.ERR_ALIGN
    assert back(dx=None, dA=None, dB=None) == back(T=0, dA=None, dB=None) == _lib.OK


@pytest.mark.gpu
def test_refusals():
    c = inputs(10, 64, 32, 8, 2, "fp16", "mixed")
    base, x, A, B, ids, s = (c[k] for k in ("base", "x", "A", "B", "ids", "scaling"))
    plan = ops.lora_plan(ids, 2)
    big = torch.zeros(400, dtype=torch.float16, device="cuda")
    for args, err in [((base, x[:, :32], A, B, plan), ValueError), ((base[:5], x, A, B, plan), ValueError),
                      ((base, x, A, B[:1], plan), ValueError), ((base, x, A, B[:, :4], plan), ValueError),
                      ((base.bfloat16(), x, A, B, plan), TypeError), ((base.float(), x.float(), A, B, plan), TypeError),
                      ((base, x, A, B, ops.lora_plan(ids, 3)), ValueError), ((base, x, A, B, ops.lora_plan(ids[:9], 2)), ValueError),
                      ((base, x, A, B, ids[None]), ValueError), ((base, x, A, B, ids.float()), ValueError),
                      ((base, x, A, B, plan, s[:1]), ValueError), ((base, x, A, B, plan, s.cpu()), ValueError),
                      ((base, x, A, B, plan, s.clone().requires_grad_()), ValueError),
                      ((base, x, A, B, plan, s, base[:, :16]), ValueError), ((base, x, A, B, plan, s, base.t()), ValueError),
                      ((base, x, A.clone().requires_grad_(), B, plan, s, base), ValueError),
                      ((base, x, A, B, plan, s, x.view(-1)[:320].view(10, 32)), ValueError),
                      ((big[:320].view(10, 32), x, A, B, plan, s, big[32:352].view(10, 32)), ValueError),
                      ((base, x[0], A, B, plan), ValueError)]:
        with pytest.raises(err):
            ops.lora_apply(*args)
    with pytest.raises(_lib.B200QError):
        ops.lora_apply(base, x, torch.zeros(2, 64, 65, device="cuda").half(), torch.zeros(2, 65, 32, device="cuda").half(), plan)
    with pytest.raises(_lib.B200QError):
        ops.lora_plan(ids, 1024)
    with pytest.raises(_lib.B200QError):
        ops.lora_plan(ids, 0)
