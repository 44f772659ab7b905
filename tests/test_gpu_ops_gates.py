"""How exact a gate is: sigmoid and its complement to a relative (1.25 |z| + 8)
2^-24 over all of f32's exponential, as the kernels state it. The error's terms:
|z| log2(e) rounded (|z| units of 2^-24 of the exponential, a quarter of that for
the constant), the exponential and the reciprocal (two units each), a sum, a
product, and the result (four at most)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from phyz_amd.ops import Ops
    return Ops(0)


def points():
    g = torch.Generator().manual_seed(0)
    z = torch.cat([torch.linspace(-85, 85, 6801), torch.randn(4000, generator=g) * 3])
    return z.clamp(-85, 85)


def test_gates_of_the_recurrence(ops):
    """From 0, one step writes 1 - sigmoid(z) of 1; a state of 1 keeps sigmoid(z)."""
    z = points()
    n, zd = z.numel(), z.double()
    room = (1.25 * zd.abs() + 8) * U
    one = torch.ones(1, 1, n, device="cuda")
    zc = z.view(1, 1, n).cuda()
    h, _ = ops.gated_scan(zc, one)
    want = torch.sigmoid(-zd)
    assert bool(((h.view(-1).cpu().double() - want).abs() <= room * want).all())
    h, _ = ops.gated_scan(zc, torch.zeros_like(one), h0=one[0])
    want = torch.sigmoid(zd)
    assert bool(((h.view(-1).cpu().double() - want).abs() <= room * want).all())


def test_gates_of_silu(ops):
    """silu(p) / p: a row of inputs through weights of 1."""
    p = points()
    pd = p.double()
    y = ops.linear(p.view(-1, 1).cuda(), torch.ones(1, 1, device="cuda"), act="silu").view(-1).cpu().double()
    want = pd * torch.sigmoid(pd)
    assert bool(((y - want).abs() <= (1.25 * pd.clamp(max=0).abs() + 9) * U * want.abs()).all())
