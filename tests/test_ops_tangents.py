"""Forward-mode tangents that would be lost are refused, on a handle without a GPU."""
import pytest
import torch
from torch.autograd import forward_ad

from phyz_amd.ops import Ops, OpsError
from tests.test_ops_autograd import FORWARD, GRADIENTS


@pytest.fixture(scope="module")
def ops():
    return Ops(device=-1)


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def dual(*shape):
    return forward_ad.make_dual(torch.zeros(shape), torch.ones(shape))


CALLS = [*FORWARD, ("x", lambda o, r: o.rotary(r(4, 2, 12), t(4, 2, dtype=torch.int64), t(2, dtype=torch.float64))),
         ("x", lambda o, r: o.rotary(r(4, 12), t(4, dtype=torch.int64), t(2, dtype=torch.float64))),
         ("k", lambda o, r: o.linear_attention(t(6, 2, 12), r(6, 2, 12), t(6, 2, 15), t(6, 2, 3))),
         ("g", lambda o, r: o.linear_attention(t(6, 2, 12), t(6, 2, 12), t(6, 2, 15), r(3))),
         ("s0", lambda o, r: o.linear_attention(t(6, 2, 12), t(6, 2, 12), t(6, 2, 15), t(6, 2, 3), s0=r(2, 3, 4, 5))),
         ("s", lambda o, r: o.linear_attention_step(t(2, 12), t(2, 12), t(2, 15), t(2, 3), r(2, 3, 4, 5)))]


@pytest.mark.parametrize("name, call", CALLS)
def test_tangents_that_would_be_lost_are_refused(ops, name, call):
    with forward_ad.dual_level():
        for quiet in (torch.enable_grad, torch.no_grad):  # which leaves tangents as they are
            with quiet(), pytest.raises(OpsError, match=f"^{name} carries a tangent"):
                call(ops, dual)
        with pytest.raises(OpsError, match="host-only"):
            call(ops, lambda *s: dual(*s).detach())
        with pytest.raises(OpsError, match="host-only"):
            call(ops, t)


@pytest.mark.parametrize("call", GRADIENTS)
def test_gradients_own_operators_take_them(ops, call):
    with forward_ad.dual_level(), pytest.raises(OpsError, match="host-only"):
        call(ops, dual)
