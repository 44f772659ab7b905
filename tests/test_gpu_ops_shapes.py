"""Shapes and views of the sequence operators at their edges, on the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from phyz_amd.ops import Ops
    return Ops(0)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_batches_without_elements(ops, dtype):
    """No features: the bias alone, and no gradient but its own. No outputs: zeros."""
    def t(*s):
        return torch.randn(*s, device="cuda").to(dtype)

    bias, dy = t(7), t(2, 4, 7)
    y = ops.linear(t(2, 4, 0), t(7, 0), bias=bias)
    assert torch.equal(y, bias.expand(2, 4, 7))
    dx, dw, db = ops.linear_backward(dy, t(2, 4, 0), t(7, 0))
    assert dx.shape == (2, 4, 0) and dw.shape == (7, 0)
    assert torch.equal(db, ops.linear_backward(dy.view(8, 7), t(8, 3), t(7, 3))[2])
    assert ops.linear(t(2, 4, 3), t(0, 3)).shape == (2, 4, 0)
    dx, dw, db = ops.linear_backward(t(2, 4, 0), t(2, 4, 3), t(0, 3))
    assert dx.shape == (2, 4, 3) and not dx.any() and dw.shape == (0, 3) and db.shape == (0,)


def test_rows_far_apart_give_the_same_bits(ops):
    """Rows 32 MiB apart, forward and backward, in inputs and in output gradients:
    strides do not change results."""
    m, k, n = 300, 64, 48
    x = torch.as_strided(torch.zeros((m - 1) * (1 << 24) + k, dtype=BF16, device="cuda"), (m, k), (1 << 24, 1))
    x.copy_(torch.randn(m, k, device="cuda"))
    w, dy = torch.randn(n, k, device="cuda").to(BF16), torch.randn(m, n, device="cuda").to(BF16)
    assert torch.equal(ops.linear(x, w), ops.linear(x.contiguous(), w))
    for a, b in zip(ops.linear_backward(dy, x, w), ops.linear_backward(dy, x.contiguous(), w)):
        assert torch.equal(a, b)
    dx = ops.linear_backward(x, dy, torch.randn(k, n, device="cuda").to(BF16), need_dx=False, need_db=False)[1]
    assert torch.equal(dx, ops.linear_backward(x.contiguous(), dy, torch.zeros(k, n, device="cuda").to(BF16), need_dx=False,
                                               need_db=False)[1])


@pytest.mark.parametrize("T, B, D", [(40, 3, 13), (600, 300, 64), (4000, 2, 33)])
def test_a_record_of_states(ops, T, B, D):
    """h0 and the states, or the states and the last one, side by side in one record
    [worlds, steps + 1, width]."""
    z, x = torch.randn(T, B, D, device="cuda"), torch.randn(T, B, D, device="cuda")
    h0 = torch.randn(B, D, device="cuda")
    h, last = ops.gated_scan(z, x, h0=h0)
    record = torch.full((B, T + 1, D), 7.0, device="cuda")
    record[:, 0] = h0
    end = torch.empty(B, D, device="cuda")
    ops.gated_scan(z, x, h0=record[:, 0], out=(record[:, 1:].transpose(0, 1), end))
    assert torch.equal(record[:, 0], h0) and torch.equal(record[:, 1:].transpose(0, 1), h) and torch.equal(end, last)
    ops.gated_scan(z, x, h0=h0, out=(record[:, :T].transpose(0, 1), record[:, T]))
    assert torch.equal(record[:, :T].transpose(0, 1), h) and torch.equal(record[:, T], last)
