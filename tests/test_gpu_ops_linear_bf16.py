"""The linear layer's gradients in bf16: rounded once, where they are stored.

Their bounds are f32's (tests/ops_ref.py) on the same inputs, 2^-16 of the
products' magnitudes for dz as the matrix cores take it, and one rounding to
bf16."""
import pytest
import torch

from tests import ops_ref as R

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
#: A row, an output, sizes on and off vectors and tiles, split sums, every path.
SHAPES = [(1, 33, 13), (1, 64, 1), (2, 361, 679), (225, 370, 1), (740, 214, 283), (64, 64, 64), (2000, 55, 9), (4096, 256, 256),
          (3001, 1024, 2056), (257, 4104, 520), (9000, 131, 1003), (2100, 1001, 2049), (70000, 64, 72)]


@pytest.fixture(scope="module")
def ops():
    from phyz_amd.ops import Ops
    return Ops(0)


def data(m, k, n, seed=0):
    g = torch.Generator().manual_seed(seed)

    def r(*s, scale=1.0):
        return (torch.randn(*s, generator=g) * scale).to("cuda", BF16)

    return r(m, n, scale=0.02), r(m, k), r(n, k, scale=k ** -0.5), r(m, n)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients_are_rounded_once(ops, shape):
    dy, x, w, pre = data(*shape)
    act = ("tanh", "silu", "gelu", "relu")[sum(shape) % 4]
    got = ops.linear_backward(dy, x, w, pre=pre, act=act)
    want, bounds = R.linear_backward(dy.float(), x.float(), w.float(), pre.float(), act, F32)
    dz = (R.d64(dy) * R.act_grad(act, R.d64(pre))).abs()
    cut = (2.0 ** -16 * dz @ R.d64(w).abs(), 2.0 ** -16 * dz.T @ R.d64(x).abs(), torch.zeros(shape[2], dtype=torch.float64))
    for name, a, b, c, e in zip(("dx", "dw", "db"), got, want, bounds, cut):
        R.within(a, b, c + e + R.U_BF16 * b.abs(), name)
    for a, b in zip(got, ops.linear_backward(dy, x, w, pre=pre, act=act)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("shape", [(1, 33, 13), (40, 96, 64), (2000, 520, 1032)], ids=str)
def test_infinite_and_nan_operands(ops, shape):
    """As f32's products have them: infinite gradients, weights and inputs, those
    times 0, and infinities of both signs."""
    m, k, n = shape
    dy, x, w, pre = data(*shape)
    inf, nan = float("inf"), float("nan")
    dy[0, 2], w[3, 5], w[4, 6] = inf, inf, -inf
    w[2, 7], x[0, 9], x[0, 10] = 0.0, inf, 0.0
    if m > 1:
        dy[1, 1], x[2, 3], dy[2, 4] = nan, -inf, 0.0
    pre.clamp_(-2, 2)
    got = ops.linear_backward(dy, x, w, pre=pre, act="silu")
    dz = R.d64(dy) * R.act_grad("silu", R.d64(pre))
    for name, a, b in (("dx", got[0], dz @ R.d64(w)), ("dw", got[1], dz.T @ R.d64(x)), ("db", got[2], dz.sum(0))):
        a = a.cpu().double()
        assert torch.equal(torch.isnan(a), torch.isnan(b)), name
        bad = torch.isinf(b)
        assert torch.equal(a[bad], b[bad]) and torch.equal(torch.isinf(a), bad), name
