"""The balance loss to the bound of the sums that its kernels make."""
import pytest
import torch

from kernelbench_harbor_b200 import ops
from tests.test_moe_balance import bounds, definition, inputs


def steps(T, E):
    """Additions that a token's probability passes through in fp32 on its way into
    the loss.  A row is split over G lanes, a warp holds 32 / G rows, a block has
    32 warps; one block up to 16384 logits, otherwise one for each step of rows
    that a block makes, 148 at most.  A lane adds its own rows, the rows of a warp
    meet in shuffles, then the 32 warps, then the blocks (1024 / EP threads an
    expert, EP the power of two that E fills, at least 8: a slice of the blocks
    each, and the slices).  The terms of E experts: 5 shuffles and 32 warps."""
    G = 1
    while 8 * G < E:
        G *= 2
    per_block = 32 * (32 // G)
    nb = 1 if T * E <= 16384 else min(-(-T // per_block), 148)
    own = -(-T // (nb * per_block))
    shuffles = (32 // G).bit_length() - 1
    EP = 8
    while EP < E:
        EP *= 2
    slices = 1024 // EP
    return own + shuffles + 32 + (-(-nb // slices) + slices if nb > 1 else 0) + 5 + 32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,E,k,masked", [
    (1, 2, 1, 0.0), (512, 8, 2, 0.25), (2048, 8, 2, 0.0), (2049, 8, 2, 0.0), (333, 17, 4, 0.5), (2049, 64, 8, 0.1),
    (1000, 256, 8, 0.3), (20000, 16, 2, 0.2), (131072, 64, 2, 0.15), (300000, 3, 1, 0.0), (40000, 256, 4, 0.0)])
def test_loss_to_the_bound_of_its_sums(T, E, k, masked, dtype):
    """Every summand is positive: each addition is off by 2^-24 of its sum at most.
    Six more for the factors (1 / n, c / n, / k, E, p / n, the product)."""
    logits, topi, mask = inputs(T, E, k, dtype, masked=masked)
    loss, counts = ops.moe_balance_loss(logits, topi, mask)
    want, wcounts, _, _ = definition(logits, topi, mask)
    assert torch.equal(counts.long(), wcounts)
    p, _ = bounds(logits, mask)  # of a probability
    assert abs(loss.double() - want) <= (p + (steps(T, E) + 6) * 2.0 ** -24) * want
