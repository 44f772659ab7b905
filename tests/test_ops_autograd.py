"""The sequence operators beside autograd, on a handle without a GPU: gradients
that would be lost are refused."""
import pytest
import torch

from phyz_amd.ops import Ops, OpsError


@pytest.fixture(scope="module")
def ops():
    return Ops(device=-1)


def t(*shape):
    return torch.zeros(*shape)


def p(*shape):
    return torch.zeros(*shape, requires_grad=True)


FORWARD = [
    ("w", lambda o, r: o.linear(t(4, 3), r(7, 3))), ("x", lambda o, r: o.linear(r(2, 4, 3), t(7, 3))),
    ("bias", lambda o, r: o.linear(t(4, 3), t(7, 3), bias=r(7))),
    ("residual", lambda o, r: o.linear(t(4, 3), t(7, 3), residual=r(4, 7))),
    ("z", lambda o, r: o.gated_scan(r(6, 2, 5), t(6, 2, 5))), ("h0", lambda o, r: o.gated_scan(t(6, 2, 5), t(6, 2, 5), h0=r(2, 5))),
    ("x", lambda o, r: o.gated_step(t(2, 5), r(2, 5), t(2, 5))), ("h", lambda o, r: o.gated_step(t(2, 5), t(2, 5), r(2, 5))),
    ("g", lambda o, r: o.orthogonalize(r(4, 5)))]
GRADIENTS = [lambda o, r: o.linear_backward(t(4, 7), t(4, 3), r(7, 3)),
             lambda o, r: o.gated_scan_backward(t(6, 2, 5), r(6, 2, 5), t(6, 2, 5), t(6, 2, 5)),
             lambda o, r: o.muon_step(r(4, 5), t(4, 5), t(4, 5))]


@pytest.mark.parametrize("name, call", FORWARD)
def test_gradients_that_would_be_lost_are_refused(ops, name, call):
    with pytest.raises(OpsError, match=f"^{name} requires gradients"):
        call(ops, p)
    for quiet in (torch.no_grad, torch.inference_mode):
        with quiet(), pytest.raises(OpsError, match="host-only"):
            call(ops, p)
    with pytest.raises(OpsError, match="host-only"):
        call(ops, lambda *s: p(*s).detach())


@pytest.mark.parametrize("call", GRADIENTS)
def test_gradients_own_operators_take_parameters(ops, call):
    with pytest.raises(OpsError, match="host-only"):
        call(ops, p)
