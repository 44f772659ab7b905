"""Rotary positions where a lane takes four pairs: many rows, pairs and sizes that
are multiples of four, rows off any alignment but their elements'."""
import pytest
import torch

from tests import attend_ref as R
from tests import test_gpu_ops_rotary as A

pytestmark = pytest.mark.gpu
ops = A.ops


@pytest.mark.parametrize("dtype", [A.F32, A.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T, B, H, size, pairs", [(64, 301, 2, 64, 32), (3, 7001, 1, 40, 12), (20001, 1, 2, 128, 64), (130, 150, 3, 32, 0)])
def test_turns(ops, T, B, H, size, pairs, layout, dtype):
    x, p, f = A.inputs(T, B, H, size, pairs, dtype, 10 ** 6, seed=size)
    want, bound = R.rotary(x, p, f, H, layout, 1.3, False)
    R.within(ops.rotary(x, p, f, heads=H, layout=layout, scale=1.3), want, bound + 1e-37, "y")
    wide = torch.full((B, T, H * size + 3), 4.0, dtype=dtype, device="cuda")
    view = wide.transpose(0, 1)[..., 1:1 + H * size]
    view.copy_(x)
    ops.rotary(view, p.int(), f, heads=H, layout=layout, scale=1.3, out=view)
    R.within(view, want, bound + 1e-37, "in place")
    assert bool((wide[..., :1] == 4).all()) and bool((wide[..., 1 + H * size:] == 4).all())


def test_many_rows_and_few_are_turned_alike(ops):
    """A step's rows, single pairs a lane, against the same rows of a rollout."""
    x, p, f = A.inputs(64, 301, 2, 64, 32, A.F32, 10 ** 6, seed=5)
    whole = ops.rotary(x, p, f, heads=2)
    for t in (0, 63):
        assert torch.equal(ops.rotary(x[t], p[t], f, heads=2), whole[t])
