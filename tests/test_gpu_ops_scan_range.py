"""The decay form where the product of many gates leaves f32's range and the
states do not: the answer is that of the steps one after the other, however
they are shared among waves and chunks (tests/ops_ref.py's bounds, element by
element)."""
import math

import pytest
import torch

from tests import ops_ref as R

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
#: One wave for all steps; waves that share slabs; chunks over the grid, of 64 to
#: 128 steps and of 512 (the state's start is a chunk's: both fold products).
SHAPES = [(600, 17000, 4), (600, 300, 64), (1100, 130, 129), (4000, 2, 33), (4099, 1, 260), (32768, 1, 8)]


@pytest.fixture(scope="module")
def ops():
    from phyz_amd.ops import Ops
    return Ops(0)


def gates(T, *runs):
    """[T] of ones, with (first step, steps, value) runs in it."""
    z = torch.ones(T)
    for at, n, v in runs:
        z[at:at + n] = v
    return z


def spread(B, D):
    """Values of different significands about 1, one a channel."""
    v = 1 + torch.arange(B * D, dtype=torch.float32).reshape(B, D) % 251 / 256
    return v * torch.where(torch.arange(B * D).reshape(B, D) % 2 == 0, 1.0, -1.0)


def both_ways(ops, z, x, start, dtype, reset=None):
    """The forward recurrence, and the same one backward in time as the gradient's:
    e_t = dh_t + c_{t+1} e_{t+1} with dh = x and dh_last = start."""
    T, B, D = x.shape
    z, x, start = z.cuda().to(dtype), x.cuda().to(dtype), start.cuda()
    h, last = ops.gated_scan(z, x, h0=start, reset=reset, form="decay")
    want, wlast, bh, bl = R.scan(z, x, start, reset, "decay", dtype)
    assert float(want.abs().max()) < 2.0 ** 127, "the case's own states leave f32"
    R.within(h, want, bh, "h")
    R.within(last, wlast, bl, "h_last")
    zb, xb = z.flip(0), x.flip(0)
    rb = None
    if reset is not None:  # the gradient stops at the step where an episode begins
        rb = reset.flip(0)
    stored = torch.randn(T, B, D, generator=torch.Generator().manual_seed(1)).cuda().to(dtype)
    got = ops.gated_scan_backward(xb, zb, xb, stored, reset=rb, dh_last=start, form="decay")
    want, bounds = R.scan_backward(xb, zb, xb, stored, None, rb, start, "decay", dtype)
    for name, a, b, c in zip(("dz", "dx", "dh0"), got, want, bounds):
        keep = b.abs() < 2.0 ** 127
        assert bool(keep.all()) or name == "dz"
        R.within(torch.where(keep, a.cpu().double(), 0.0), torch.where(keep, b, 0.0), c, name)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("case", ["up and down", "down and up", "up", "up, then zero gates"])
def test_products_beyond_f32(ops, case, shape, dtype):
    T, B, D = shape
    at = 5  # inside the first chunk, and (mirrored) inside the backward's first
    if case == "up and down":      # product to 2^150 on a state of 2^-40, and back
        z, size = gates(T, (at, 150, 2.0), (at + 150, 150, 0.5)), 2.0 ** -40
    elif case == "down and up":    # product to 2^-200 on a state of 2^100, and back
        z, size = gates(T, (at, 200, 0.5), (at + 200, 200, 2.0)), 2.0 ** 100
    elif case == "up":             # 3^90 = 2^142 on a state of 2^-33
        z, size = gates(T, (at, 90, 3.0), (at + 90, T - at - 90, 0.75)), 2.0 ** -33
    else:
        z, size = gates(T, (at, 150, 2.0), (at + 170, 1, 0.0), (at + 300, 20, 0.5)), 2.0 ** -40
    z = z[:, None, None].expand(T, B, D).contiguous()
    if B * D > 20000:  # many equal channels: compare some of them
        B2 = 2
        start = size * spread(B2, D)
        keep = ops.gated_scan(z.cuda().to(dtype), torch.zeros(T, B, D, device="cuda", dtype=dtype),
                              h0=start.repeat(B // B2, 1).cuda(), form="decay")
        want, wlast, bh, bl = R.scan(z[:, :B2].to(dtype), torch.zeros(T, B2, D, dtype=dtype), start, None, "decay", dtype)
        R.within(keep[0][:, :B2], want, bh, "h")
        R.within(keep[1][-B2:], wlast, bl, "h_last")
        return
    x = torch.zeros(T, B, D)
    x[at + 310 if T > 600 else T - 1] = spread(B, D)
    both_ways(ops, z, x, size * spread(B, D), dtype)


@pytest.mark.parametrize("shape", SHAPES[1:], ids=str)
def test_products_beyond_f32_within_a_few_steps(ops, shape):
    """Gates of 2^50 and 2^-50 next to each other: a run of eight steps already
    leaves f32's range either way."""
    T, B, D = shape
    z = torch.ones(T)
    z[3:9] = torch.tensor([2.0 ** 50] * 3 + [2.0 ** -50] * 3)      # 2^150 on 2^-60
    z[33:43] = torch.tensor([2.0 ** 50] * 3 + [2.0 ** -50] * 4 + [2.0 ** 50, 1.5, 1.0])
    z = z[:, None, None].expand(T, B, D).contiguous()
    both_ways(ops, z, torch.zeros(T, B, D), 2.0 ** -60 * spread(B, D), F32)


@pytest.mark.parametrize("shape", SHAPES[1:], ids=str)
def test_resets_among_growing_gates(ops, shape):
    T, B, D = shape
    reset = torch.zeros(T, B, dtype=torch.bool, device="cuda")
    reset[200], reset[T - 40] = True, True
    z = gates(T, (2, 140, 2.0), (150, 300, 0.5), (T - 60, 60, 2.0))[:, None, None].expand(T, B, D).contiguous()
    x = torch.zeros(T, B, D)
    x[210], x[T - 30] = spread(B, D), spread(B, D)
    both_ways(ops, z, x, 2.0 ** -40 * spread(B, D), F32, reset=reset)


@pytest.mark.parametrize("shape", [(600, 300, 64), (1100, 130, 129), (32768, 1, 8)], ids=str)
def test_states_that_stay_while_sums_from_zero_do_not(ops, shape):
    """h = 2 h - 1 from 1 stays 1, exactly; from 0 the 512 steps of a chunk pass
    f32's range. (Chunks of fewer steps stay in range and give what a sum of terms
    of 2^96 can: no bound of such a recurrence says more.)"""
    T, B, D = shape
    z = torch.full((T, B, D), 2.0, device="cuda")
    x = torch.full((T, B, D), -1.0, device="cuda")
    one = torch.ones(B, D, device="cuda")
    h, last = ops.gated_scan(z, x, h0=one, form="decay")
    assert torch.equal(h, torch.ones_like(h)) and torch.equal(last, one)
    # e_t = 1 + (-1 from the step after, times 2): from dh_last = -2, e = -1 throughout.
    dz, dx, dh0 = ops.gated_scan_backward(torch.ones_like(x), z, x, h, dh_last=-2 * one, form="decay")
    assert torch.equal(dx, -torch.ones_like(dx)) and torch.equal(dh0, -2 * one)


@pytest.mark.parametrize("shape", SHAPES[1:], ids=str)
def test_an_infinite_gate(ops, shape):
    """It makes of a state its infinity, not NaN, until the next episode."""
    T, B, D = shape
    z = torch.full((T, B, D), 0.5, device="cuda")
    z[100] = math.inf
    reset = torch.zeros(T, B, dtype=torch.bool, device="cuda")
    reset[T - 20] = True
    start = spread(B, D).cuda() * 2.0 ** 110  # still far from 0 at step 100
    h, _ = ops.gated_scan(z, torch.zeros_like(z), h0=start, reset=reset, form="decay")
    assert torch.equal(h[100:T - 20], (torch.sign(start) * math.inf)[None].expand(T - 120, B, D))
    assert torch.isfinite(h[:100]).all() and not h[T - 20:].any()


def test_diverged_channels_leave_the_others_alone(ops):
    """A channel that overflows by itself is infinite; the ones beside it, in the
    same lane and wave, keep their bits."""
    for T, B, D in SHAPES[1:]:
        g = torch.Generator().manual_seed(5)
        z = torch.sigmoid(torch.randn(T, B, D, generator=g)).cuda()
        x = torch.randn(T, B, D, generator=g).cuda()
        clean, cl = ops.gated_scan(z, x, form="decay")
        z2 = z.clone()
        z2[:, B // 2, 1] = 2.0
        h, last = ops.gated_scan(z2, x, form="decay")
        assert torch.isinf(h[300:, B // 2, 1]).all() and torch.isinf(last[B // 2, 1])
        h[:, B // 2, 1], last[B // 2, 1] = clean[:, B // 2, 1], cl[B // 2, 1]
        assert torch.equal(h, clean) and torch.equal(last, cl)


def test_zero_states_pass_chunks_of_growing_gates(ops):
    """A state of 0 under chunks of 512 gates of 2, of which the product is 2^512."""
    shape = (32768, 1, 8)
    z, x = torch.full(shape, 2.0, device="cuda"), torch.zeros(shape, device="cuda")
    x[-1] = 3.0
    h, last = ops.gated_scan(z, x, form="decay")
    assert not h[:-1].any() and bool((h[-1] == 3).all()) and bool((last == 3).all())
    dz, dx, dh0 = ops.gated_scan_backward(x.flip(0), z, x, h, form="decay")
    assert not dx[1:].any() and bool((dx[0] == 3).all()) and bool((dh0 == 6).all())
