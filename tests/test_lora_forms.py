"""The one-launch form and the tiled pair where one hands over to the other."""
import pytest
import torch

from kernelbench_harbor_b200 import ops
from tests.test_lora_apply import check, close, inputs, pair


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("r", [32, 33, 40, 64])
@pytest.mark.parametrize("T,D,N", [(128, 256, 264), (129, 256, 264), (200, 99, 130), (256, 264, 128), (257, 264, 128)])
def test_around_the_handover(T, D, N, r, dtype):
    c = inputs(T, D, N, r, 3, dtype, "runs")
    y, _ = check(c)
    with torch.no_grad():  # the same form with and without a gradient
        assert torch.equal(ops.lora_apply(c["base"], c["x"], c["A"], c["B"], c["ids"], c["scaling"]), y)


@pytest.mark.gpu
def test_without_room_for_the_row_between():
    """The C entry takes lo = NULL up to 256 tokens at every rank."""
    from kernelbench_harbor_b200 import _lib
    for T in (129, 256):
        c = inputs(T, 256, 264, 64, 3, "bf16", "runs")
        plan, y = ops.lora_plan(c["ids"], 3), torch.empty_like(c["base"])
        _lib.check(_lib.lib().b200q_lora_apply(
            c["x"].data_ptr(), c["base"].data_ptr(), c["A"].data_ptr(), c["B"].data_ptr(), c["scaling"].data_ptr(),
            plan.data.data_ptr(), T, 256, 264, 64, 3, _lib.DTYPE_BF16, y.data_ptr(), None, None,
            torch.cuda.current_stream().cuda_stream))
        _, want, _, err = pair(c["x"], c["A"], c["B"], c["scaling"], c["ids"], c["base"])
        close(y, want, err, torch.bfloat16)
