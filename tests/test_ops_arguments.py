"""Arguments of the sequence operators at their edges, on a handle without a
GPU: what is right reaches the device check, what is not is named."""
import pytest
import torch

from phyz_amd.ops import Ops, OpsError

F32 = torch.float32


@pytest.fixture(scope="module")
def ops():
    return Ops(device=-1)


def t(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call", [
    lambda o: o.linear(t(2, 4, 0), t(7, 0), bias=t(7)),
    lambda o: o.linear(t(0, 4, 3), t(7, 3)),
    lambda o: o.linear(t(2, 4, 3), t(0, 3), residual=t(2, 4, 0)),
    lambda o: o.linear_backward(t(2, 4, 7), t(2, 4, 0), t(7, 0)),
    lambda o: o.linear_backward(t(2, 4, 0), t(2, 4, 3), t(0, 3)),
], ids=["no features", "no rows", "no outputs", "no features, backward", "no outputs, backward"])
def test_batches_without_elements(ops, call):
    """As their two-dimensional forms: right, and only then without a device."""
    with pytest.raises(OpsError, match="host-only"):
        call(ops)
