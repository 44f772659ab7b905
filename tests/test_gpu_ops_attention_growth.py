"""Gates above 0, as far as they are documented: states that grow 2^32-fold in 16
steps, and what they come to again where the gates close."""
import math

import pytest
import torch

from tests import test_gpu_ops_attention as A

pytestmark = pytest.mark.gpu
ops = A.ops
DOUBLE = math.log(2.0)
# Of a period of steps: how many grow, and by how much each; the others take it back.
PERIODS = {"16 up, 16 down": (32, 16, 2 * DOUBLE), "1 up, 20 down": (21, 1, 32 * DOUBLE), "48 up, 48 down": (96, 48, 2 * DOUBLE),
           "5 up, 90 down": (95, 5, 6.4 * DOUBLE)}


@pytest.mark.parametrize("dtype", [A.F32, A.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("period", PERIODS)
@pytest.mark.parametrize("phase", [0, 9])
# One chunk, several, and segments of them.
@pytest.mark.parametrize("T, B, H, nk, nv", [(30, 2, 2, 16, 24), (200, 2, 2, 32, 40), (1500, 1, 1, 64, 64)])
def test_gates_that_grow_and_close(ops, T, B, H, nk, nv, phase, period, dtype):
    n, up, by = PERIODS[period]
    x = A.inputs(T, B, H, nk, nv, dtype, 31, reset=0.002)
    at = (torch.arange(T, device="cuda") + phase) % n
    x["g"] = torch.where(at < up, by, -by * up / (n - up)).float()[:, None, None].expand(T, B, H).contiguous()
    A.check_forward(A.forward(ops, x, nk, nv), x, nk, nv)
    A.check_backward(A.backward(ops, x, nk, nv), x, nk, nv)
