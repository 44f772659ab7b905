"""Linear attention where waves have no columns, workgroups are no multiple of what
goes to the chiplets together, and steps are split into uneven segments."""
import pytest
import torch

from tests import test_gpu_ops_attention as A

pytestmark = pytest.mark.gpu
ops = A.ops
# A wave has 16 columns of a head padded to 32, 64 or 128; 128 workgroups are dealt
# out together; segments have 4 chunks of 32 (f32) or 64 steps at least, the last of
# them fewer.
SIZES = [(200, 3, 5, 40, 72), (65, 27, 5, 100, 20), (130, 7, 3, 33, 65), (64, 131, 1, 16, 16), (520, 1, 2, 72, 40),
         (130, 2, 64, 20, 130 - 2), (1500, 1, 3, 17, 97), (2100, 1, 1, 128, 128), (640, 1, 1, 8, 120)]


@pytest.mark.parametrize("dtype", [A.F32, A.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T, B, H, nk, nv", SIZES)
def test_forward_and_backward(ops, T, B, H, nk, nv, dtype):
    x = A.inputs(T, B, H, nk, nv, dtype, seed=T + nk + nv)
    A.check_forward(A.forward(ops, x, nk, nv), x, nk, nv)
    A.check_backward(A.backward(ops, x, nk, nv), x, nk, nv)


@pytest.mark.parametrize("dtype", [A.F32, A.BF16], ids=["f32", "bf16"])
def test_results_do_not_depend_on_layout_or_neighbours(ops, dtype):
    """A world alone, and among others in batch-major rows that begin off any line."""
    T, B, H, nk, nv = 300, 37, 3, 24, 40
    x = A.inputs(T, B, H, nk, nv, dtype, seed=1, batch_first=True)
    o, s = A.forward(ops, x, nk, nv)
    grads = A.backward(ops, x, nk, nv)
    wide = {}
    for k in ("q", "k", "v", "do"):
        room = torch.full((T, B, x[k].shape[-1] + 5), 7.0, device="cuda", dtype=dtype)
        wide[k] = room[..., 3:3 + x[k].shape[-1]]
        wide[k].copy_(x[k])
    y = {**x, **wide}
    o2, s2 = A.forward(ops, y, nk, nv)
    assert torch.equal(o, o2) and torch.equal(s, s2)
    for a, b in zip(grads, A.backward(ops, y, nk, nv)):
        assert torch.equal(a, b)
