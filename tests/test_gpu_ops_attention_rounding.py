"""Linear attention in bf16: outputs are the rounding of what 32 bits find, not of
what fewer hold."""
import math

import pytest
import torch

from tests import attend_ref as R
from tests import test_gpu_ops_attention as A

pytestmark = pytest.mark.gpu
ops = A.ops


def from_the_rounding(got, want, terms, what):
    """The norm of got - bf16(want), in want's. n additions in 32 bits, each off by up
    to U = 2^-24 of a partial sum of the result's size, evenly spread, leave e =
    sqrt(n / 3) U of it. A value that is e off rounds to a neighbour where a midpoint
    between two bf16 is that close: in e / s of all places, s a bf16 step of 2^-8 to
    2^-7 of the value, and is s off there. That comes to e s <= 2^-7 e in the square;
    operands of two bf16 pieces (2^-17 of each) leave some ten times e and three times
    the norm."""
    want = want.float()  # 64 to 32 bits first: 2^-24, less than e
    got, near = got.cpu().double(), want.to(torch.bfloat16).double()
    off = float((got - near).norm() / near.norm())
    most = math.sqrt(math.sqrt(terms / 3) * R.U32 * 2.0 ** -7)
    assert off <= most, f"{what}: {off:.3g}, more than {most:.3g}"


@pytest.mark.parametrize("T, B, H, nk, nv", [(700, 2, 2, 64, 64), (200, 3, 5, 40, 72), (300, 2, 2, 128, 128), (2100, 1, 2, 128, 32),
                                             (520, 1, 4, 32, 128)])
def test_outputs_round_once(ops, T, B, H, nk, nv):
    x = A.inputs(T, B, H, nk, nv, A.BF16, seed=T + nk, reset=0.01)
    n = R._terms(T, nk, nv)
    (o, _), _ = R.attention(x["q"], x["k"], x["v"], x["g"], x["s0"], x["reset"], nk, nv, nk ** -0.5)
    from_the_rounding(A.forward(ops, x, nk, nv)[0], o, n, "o")
    want, _ = R.attention_backward(x["do"], x["q"], x["k"], x["v"], x["g"], x["s0"], x["reset"], x["ds"], nk, nv, nk ** -0.5)
    for got, w, what in zip(A.backward(ops, x, nk, nv), want, ("dq", "dk", "dv")):
        from_the_rounding(got, w, n, what)
