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


@pytest.mark.parametrize("call, message", [
    (lambda o: torch.vmap(lambda z: o.gated_scan(z, z))(t(3, 6, 2, 5)), "z has no strided memory"),
    (lambda o: torch.vmap(lambda z: o.gated_step(z, z, t(2, 5)))(t(3, 2, 5)), "z has no strided memory"),
    (lambda o: torch.vmap(lambda x: o.linear(x, t(7, 3)))(t(3, 4, 3)), "x has no strided memory"),
    (lambda o: o.gated_scan(t(6, 2, 5).to_sparse(), t(6, 2, 5)), "z has no strided memory"),
    (lambda o: o.gated_scan(t(()), t(())), "z has 0 dimensions, expected 1 to 3"),
    (lambda o: o.linear(t(()), t(7, 3)), "x has 0 dimensions, expected 2 or more"),
    (lambda o: o.linear(t(3), t(7, 3)), "x has 1 dimensions, expected 2 or more"),
    (lambda o: o.linear_backward(t(4, 7), t(4, 3), t(3)), "w has 1 dimensions, expected 2"),
    (lambda o: o.linear_backward(t(4, 7), t(4, 3), t(())), "w has 0 dimensions, expected 2"),
])
def test_refusals_name_the_reason(ops, call, message):
    with pytest.raises(OpsError, match=message):
        call(ops)


@pytest.mark.parametrize("rows, cols", [(32769, 1), (1, (1 << 20) + 1), (32768, 32769)])
def test_limits_of_a_matrix_are_named(ops, rows, cols):
    g = t(1, 1).expand(rows, cols)
    with pytest.raises(OpsError, match=f"g is {rows} x {cols}: at most 32768 rows, 2\\^20 columns and 2\\^30 elements"):
        ops.orthogonalize(g, out=g)
