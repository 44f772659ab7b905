"""The sigmoid form where states and inputs are near f32's largest number: their
differences are not in range, the states are."""
import pytest
import torch

from tests import ops_ref as R

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from phyz_amd.ops import Ops
    return Ops(0)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 5, 7), (40, 3, 9), (600, 300, 64), (4000, 2, 33)], ids=str)
def test_differences_beyond_f32(ops, shape, dtype):
    """A state is a mean of inputs, whatever their size and signs; and so the
    gradients for gates, with output gradients of 1e-8."""
    g = torch.Generator().manual_seed(1)
    T, B, D = shape
    big = 3.3e38
    z = torch.randn(T, B, D, generator=g) * 3
    x = torch.where(torch.rand(T, B, D, generator=g) < 0.5, -big, big)
    h0 = torch.where(torch.rand(B, D, generator=g) < 0.5, -big, big).cuda()
    z, x = z.cuda().to(dtype), x.cuda().to(dtype)
    h, last = ops.gated_scan(z, x, h0=h0)
    want, wlast, bh, bl = R.scan(z, x, h0, None, "sigmoid", dtype)
    R.within(h, want, bh, "h")
    R.within(last, wlast, bl, "h_last")
    if T == 1:
        s = h0.clone()
        ops.gated_step(z[0], x[0], s)
        R.within(s, wlast, bl, "step")
    dh = (torch.randn(T, B, D, generator=g) * 1e-8).cuda().to(dtype)
    got = ops.gated_scan_backward(dh, z, x, h, h0=h0)
    want, bounds = R.scan_backward(dh, z, x, h, h0, None, None, "sigmoid", dtype)
    for name, a, b, c in zip(("dz", "dx", "dh0"), got, want, bounds):
        R.within(a, b, c, name)
