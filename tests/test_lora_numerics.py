"""Adapters in fp16 where values of very different sizes share a row or an
adapter: a large one must not cost the small ones their bits."""
import pytest
import torch

from kernelbench_harbor_b200 import ops
from tests.test_lora_apply import STEP, close, inputs, pair

FLOOR = 2.0 ** -39  # of the largest value that is scaled together with a value: the halves' smallest step
SPLIT = 2.0 ** -22  # two fp16 halves of a value: half a step of half a step


def expand(base, mid, emid, Q, ids):
    """(y, its error bound before the last rounding) of base + mid . Q[id] in float64."""
    out, err = base.double().clone(), torch.zeros(base.shape, dtype=torch.float64, device=base.device)
    for a in range(Q.shape[0]):
        t = torch.nonzero(ids == a).flatten()
        m, q = mid[t], Q[a].double()
        e = emid[t] + SPLIT * m.abs() + FLOOR * m.abs().amax(dim=1, keepdim=True) if len(t) else emid[t]
        out[t] += m @ q
        err[t] = e @ q.abs() + (Q.shape[1] / 16 + 4) * STEP * (m.abs() @ q.abs()) + STEP * out[t].abs()
    return out, err


def sums(wide, thin, ethin, ids, L):
    """(sum_t wide^T thin per adapter, its error bound before the last rounding)."""
    W = wide.double()
    out = torch.zeros(L, W.shape[1], thin.shape[1], dtype=torch.float64, device=W.device)
    err = torch.zeros_like(out)
    for a in range(L):
        t = torch.nonzero(ids == a).flatten()
        if not len(t):
            continue
        w, m = W[t], thin[t]
        e = ethin[t] + SPLIT * m.abs() + FLOOR * m.abs().max()
        out[a] = w.t() @ m
        err[a] = w.abs().t() @ e + (len(t) / 16 + 48) * STEP * (w.abs().t() @ m.abs())
    return out, err


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,N,r,L", [(40, 128, 96, 8, 1), (200, 128, 96, 33, 2), (700, 136, 256, 16, 2), (700, 130, 99, 5, 2),
                                       (600, 128, 264, 64, 1), (9000, 128, 128, 64, 1), (3000, 256, 512, 40, 2)])
@pytest.mark.parametrize("gap", [16, 20])
def test_one_large_token_in_fp16(T, D, N, r, L, gap):
    """One token of each adapter whose output gradient, and whose row between, are
    2^gap times the others', with x and dy zero in the first half of their
    columns: there, dA and dB are the other tokens' sums alone."""
    c = inputs(T, D, N, r, L, "fp16", "mixed")
    c["scaling"].fill_(1.0)
    big = torch.tensor([int(torch.nonzero(c["ids"] == a).flatten()[0]) for a in range(L)], device="cuda")
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[big] = False
    # the others small, the one large: the products of two halves of the gap each
    for name, half in (("x", D // 2), ("dy", N // 2)):
        v = c[name].float()
        v[rest] *= 2.0 ** -(gap // 2)
        v[big] *= 2.0 ** (gap - gap // 2)
        v[big, :half] = 0
        c[name] = v.half()
    leaves = [c[k].clone().requires_grad_() for k in ("x", "A", "B")]
    y = ops.lora_apply(c["base"], *leaves, c["ids"], c["scaling"])
    dx, dA, dB = torch.autograd.grad(y, leaves, c["dy"])
    lo, _, elo, _ = pair(c["x"], c["A"], c["B"], c["scaling"], c["ids"])
    dlo, _, edlo, _ = pair(c["dy"], c["B"].transpose(1, 2), c["A"].transpose(1, 2), c["scaling"], c["ids"])
    close(dA, *sums(c["x"], dlo, edlo, c["ids"], L), torch.float16)
    wB, eB = sums(c["dy"], lo, elo, c["ids"], L)
    close(dB, wB.transpose(1, 2), eB.transpose(1, 2), torch.float16)
    close(y.detach(), *expand(c["base"], lo, elo, c["B"], c["ids"]), torch.float16)
    close(dx, *expand(torch.zeros_like(c["x"]), dlo, edlo, c["A"].transpose(1, 2), c["ids"]), torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,N,r", [(1, 64, 96, 8), (40, 128, 96, 16), (40, 120, 99, 33), (700, 136, 256, 16), (700, 130, 99, 5),
                                     (600, 128, 264, 64), (9000, 128, 128, 64)])
@pytest.mark.parametrize("gap", [16, 22])
def test_one_large_rank_in_fp16(T, D, N, r, gap):
    """The first rank's lo (dlo) is 2^gap times the others' and its row of B (column
    of A) zero in the first half: there y (dx) is the other ranks' alone."""
    c = inputs(T, D, N, r, 1, "fp16", "one")
    c["scaling"].fill_(1.0)
    c["base"].zero_()
    up, down = 2.0 ** (gap - gap // 2), 2.0 ** -(gap // 2)

    def sized(t, rank):  # 2^gap between the first rank and the others
        v = t.float() * down
        v.select(rank, 0).mul_(up / down)
        return v.half()

    A, B = sized(c["A"], 2), c["B"].clone()
    B[:, 0, :N // 2] = 0
    y = ops.lora_apply(c["base"], c["x"], A, B, c["ids"], c["scaling"])
    lo, _, elo, _ = pair(c["x"], A, B, c["scaling"], c["ids"])
    close(y, *expand(c["base"], lo, elo, B, c["ids"]), torch.float16)

    A, B = c["A"].clone(), sized(c["B"], 1)
    A[:, :D // 2, 0] = 0
    x = c["x"].clone().requires_grad_()
    (dx,) = torch.autograd.grad(ops.lora_apply(c["base"], x, A, B, c["ids"], c["scaling"]), x, c["dy"])
    dlo, _, edlo, _ = pair(c["dy"], B.transpose(1, 2), A.transpose(1, 2), c["scaling"], c["ids"])
    close(dx, *expand(torch.zeros_like(x), dlo, edlo, A.transpose(1, 2), c["ids"]), torch.float16)
