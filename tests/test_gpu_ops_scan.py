"""The gated linear recurrence on the device against 64 bits, element by
element within bounds of its arithmetic (tests/ops_ref.py)."""
import pytest
import torch

from tests import ops_ref as R

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
#: steps, worlds, width: one step, one channel, widths below and off the vector
#: of four, runs and slabs that end off their sizes, a chunked long sequence,
#: and many worlds.
SHAPES = [(1, 1, 1), (1, 7, 33), (2, 3, 3), (5, 2, 4), (17, 3, 129), (64, 2, 64), (65, 5, 7), (257, 1, 2), (300, 3, 70),
          (1000, 1, 256), (4099, 2, 37), (33, 700, 5), (9, 1500, 260), (2050, 1, 8)]


@pytest.fixture(scope="module")
def ops():
    from phyz_amd.ops import Ops
    return Ops(0)


def data(T, B, D, dtype, form, seed=0, reset=True, batch_first=False):
    g = torch.Generator().manual_seed(seed)

    def lay(v):
        v = v.to("cuda", dtype)
        return v.transpose(0, 1).contiguous().transpose(0, 1) if batch_first else v

    def n(*s):
        return torch.randn(*s, generator=g)

    z = n(T, B, D) * 2 + 1
    if form == "decay":
        z = torch.sigmoid(z) * torch.where(torch.rand(T, B, D, generator=g) < 0.1, -1.0, 1.0)
    d = {"z": lay(z), "x": lay(n(T, B, D)), "h0": n(B, D).cuda(), "dh": lay(n(T, B, D)), "h": lay(n(T, B, D)),
         "dh_last": n(B, D).cuda()}
    d["reset"] = (torch.rand(T, B, generator=g) < 0.1).cuda() if reset else None
    return d


@pytest.mark.parametrize("form", ["sigmoid", "decay"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(ops, shape, dtype, form):
    d = data(*shape, dtype, form, reset=sum(shape) % 2 == 0, batch_first=sum(shape) % 3 == 0)
    h, last = ops.gated_scan(d["z"], d["x"], h0=d["h0"], reset=d["reset"], form=form)
    want, wlast, bh, bl = R.scan(d["z"], d["x"], d["h0"], d["reset"], form, dtype)
    R.within(h, want, bh, "h")
    R.within(last, wlast, bl + 1e-30, "h_last")
    got = ops.gated_scan_backward(d["dh"], d["z"], d["x"], d["h"], h0=d["h0"], reset=d["reset"], dh_last=d["dh_last"],
                                  form=form)
    want, bounds = R.scan_backward(d["dh"], d["z"], d["x"], d["h"], d["h0"], d["reset"], d["dh_last"], form, dtype)
    for name, a, b, c in zip(("dz", "dx", "dh0"), got, want, bounds):
        R.within(a, b, c, name)
    if shape[0] == 1:
        s = d["h0"].clone()
        assert ops.gated_step(d["z"][0], d["x"][0], s, reset=None if d["reset"] is None else d["reset"][0],
                              form=form) is s
        R.within(s, wlast, bl + 1e-30, "step")


def test_optional_arguments_are_zeros(ops):
    d = data(40, 3, 20, F32, "sigmoid", reset=False)
    zero = torch.zeros(3, 20, device="cuda")
    a = ops.gated_scan(d["z"], d["x"])
    b = ops.gated_scan(d["z"], d["x"], h0=zero, reset=torch.zeros(40, 3, dtype=torch.uint8, device="cuda"))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    a = ops.gated_scan_backward(d["dh"], d["z"], d["x"], d["h"])
    b = ops.gated_scan_backward(d["dh"], d["z"], d["x"], d["h"], h0=zero, dh_last=zero)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("form", ["sigmoid", "decay"])
@pytest.mark.parametrize("T", [1, 3, 70, 3000])
def test_reset_forgets_infinite_and_nan_states(ops, T, form):
    """Whatever an episode left behind, infinite or NaN, the next one starts at 0;
    an episode's own NaN stays in it."""
    d = data(T, 3, 9, F32, form, reset=False)
    h0 = d["h0"].clone()
    h0[0], h0[1] = float("inf"), float("nan")
    reset = torch.zeros(T, 3, dtype=torch.bool, device="cuda")
    reset[0] = True
    if T > 2:
        d["x"][T // 3, 2, 4] = float("nan")
        reset[2 * T // 3, 2] = True
    h, last = ops.gated_scan(d["z"], d["x"], h0=h0, reset=reset, form=form)
    clean = d["x"].clone()
    clean[torch.isnan(clean)] = 0.0
    want, wlast, bh, _ = R.scan(d["z"], clean, None, reset, form, F32)
    bad = torch.zeros(T, 3, 9, dtype=torch.bool)
    if T > 2:
        bad[T // 3:2 * T // 3, 2, 4] = True
    h = h.cpu()
    assert torch.isnan(h[bad]).all()
    R.within(torch.where(bad, 0.0, h), torch.where(bad, 0.0, want), bh, "h")
    # Backward: an infinite stored state before an episode's first step reaches nothing.
    hs = d["h"].clone()
    if T > 2:
        reset[T // 2] = True
        hs[T // 2 - 1] = float("inf")
    got = ops.gated_scan_backward(d["dh"], d["z"], clean, hs, h0=h0, reset=reset, form=form)
    hs[torch.isinf(hs)] = 0.0
    want, bounds = R.scan_backward(d["dh"], d["z"], clean, hs, None, reset, None, form, F32)
    for name, a, b, c in zip(("dz", "dx", "dh0"), got, want, bounds):
        R.within(a, b, c, name)
    assert torch.equal(got[2], torch.zeros_like(got[2]))


@pytest.mark.parametrize("T", [4, 900])
def test_saturated_gates(ops, T):
    """Gates at the ends of f32 keep or write exactly; within one run of steps a
    state at its value stays at it whatever the gate."""
    x = torch.randn(T, 2, 8, device="cuda")
    h0 = torch.randn(2, 8, device="cuda")
    for z, want in ((1e30, h0[None].expand(T, 2, 8)), (-1e30, x), (float("-inf"), x)):
        h, last = ops.gated_scan(torch.full_like(x, z), x, h0=h0)
        assert torch.equal(h, want) and torch.equal(last, want[-1])
    if T <= 8:
        h, _ = ops.gated_scan(torch.full_like(x, 8.0), torch.full_like(x, 0.3), h0=torch.full_like(h0, 0.3))
        assert torch.equal(h, torch.full_like(x, 0.3))


@pytest.mark.parametrize("shape", [(600, 1, 64), (600, 300, 64), (4000, 2, 33)], ids=str)
def test_zero_states_pass_growing_gates(ops, shape):
    """Gates of 2 over hundreds of steps, of which the product is past f32: a
    state of 0 stays 0, and what enters late grows exactly."""
    z, x = torch.full(shape, 2.0, device="cuda"), torch.zeros(shape, device="cuda")
    want, tail = torch.zeros(shape, device="cuda"), torch.tensor([1.0, 3.0, 7.0], device="cuda")[:, None, None]
    x[-3:], want[-3:] = 1.0, tail
    h, last = ops.gated_scan(z, x, form="decay")
    assert torch.equal(h, want) and torch.equal(last, want[-1])
    dh = x.flip(0)
    dz, dx, dh0 = ops.gated_scan_backward(dh, z, x, h, form="decay")
    assert torch.equal(dx, want.flip(0)) and not dz.any() and torch.equal(dh0, 2 * want[-1])


def test_empty(ops):
    z = torch.zeros(0, 3, 5, device="cuda")
    h0 = torch.randn(3, 5, device="cuda")
    h, last = ops.gated_scan(z, z, h0=h0)
    assert h.shape == (0, 3, 5) and torch.equal(last, h0)
    assert torch.equal(ops.gated_scan(z, z)[1], torch.zeros_like(h0))
    dz, dx, dh0 = ops.gated_scan_backward(z, z, z, z, dh_last=h0)
    assert torch.equal(dh0, h0)
    for shape in ((4, 0, 5), (4, 3, 0)):
        z = torch.zeros(shape, device="cuda")
        assert ops.gated_scan(z, z)[0].shape == shape
        ops.gated_scan_backward(z, z, z, z)


def test_halves_of_one_buffer(ops):
    """Gates and values, and their gradients, as halves of one projection."""
    T, B, D = 50, 3, 21
    both = torch.randn(T, B, 2 * D, device="cuda").to(BF16)
    z, x = both[..., :D], both[..., D:]
    h, last = ops.gated_scan(z, x)
    h2, last2 = ops.gated_scan(z.contiguous(), x.contiguous())
    assert torch.equal(h, h2) and torch.equal(last, last2)
    dh = torch.randn_like(h)
    grads = torch.full_like(both, 7.0)
    dh0 = torch.empty(B, D, device="cuda")
    ops.gated_scan_backward(dh, z, x, h, out=(grads[..., :D], grads[..., D:], dh0))
    dz, dx, dh02 = ops.gated_scan_backward(dh, z.contiguous(), x.contiguous(), h)
    assert torch.equal(grads, torch.cat([dz, dx], -1)) and torch.equal(dh0, dh02)


def test_outputs_leave_their_surroundings(ops):
    """Odd widths inside wider rows: nothing beside the view is written."""
    T, B, D = 130, 2, 13
    x = torch.randn(T, B, D, device="cuda")
    h = torch.full((T, B, 32), 5.0, device="cuda")
    last = torch.full((B, 32), 5.0, device="cuda")
    ops.gated_scan(x, x, out=(h[..., 3:3 + D], last[:, 1:1 + D]))
    want, wlast = ops.gated_scan(x, x)
    assert torch.equal(h[..., 3:3 + D], want) and torch.equal(last[:, 1:1 + D], wlast)
    h[..., 3:3 + D], last[:, 1:1 + D] = 5.0, 5.0
    assert (h == 5).all() and (last == 5).all()


def test_offsets_beyond_32_bits(ops):
    """A history whose steps lie 3 GiB apart, as slices of a long record do."""
    T, B, D = 3, 2, 5
    pitch = 3 << 29  # elements of bf16
    big = torch.empty(pitch * (T - 1) + B * D, dtype=BF16, device="cuda")
    z = torch.as_strided(big, (T, B, D), (pitch, D, 1))
    x = torch.randn(T, B, D, device="cuda").to(BF16)
    z.copy_(torch.randn(T, B, D, device="cuda"))
    h, last = ops.gated_scan(z, x)
    h2, last2 = ops.gated_scan(z.contiguous(), x)
    assert torch.equal(h, h2) and torch.equal(last, last2)


def test_scan_equals_its_steps_and_repeats(ops):
    d = data(200, 2, 40, F32, "sigmoid")
    h, last = ops.gated_scan(d["z"], d["x"], h0=d["h0"], reset=d["reset"])
    want, _, bound, _ = R.scan(d["z"], d["x"], d["h0"], d["reset"], "sigmoid", F32)
    s = d["h0"].clone()
    for t in range(200):
        ops.gated_step(d["z"][t], d["x"][t], s, reset=d["reset"][t])
        assert float(((s - h[t]).abs().cpu().double() / (2 * bound[t] + 1e-30)).max()) <= 1
    for _ in range(3):
        again = ops.gated_scan(d["z"], d["x"], h0=d["h0"], reset=d["reset"])
        assert torch.equal(again[0], h) and torch.equal(again[1], last)


@pytest.mark.parametrize("form", ["sigmoid", "decay"])
def test_gradient_against_differences(ops, form):
    """The loss's central difference along a direction, from the forward kernel,
    against the gradients' inner product with it. A difference of step s is off
    by s^2 of third derivatives and U32 |L| / s of rounding: 1e-3 covers both."""
    d = data(60, 3, 17, F32, form, seed=3)
    gen = torch.Generator().manual_seed(9)
    dirs = {k: torch.randn(d[k].shape, generator=gen).cuda() for k in ("z", "x", "h0")}
    s = 2e-3

    def loss(sign):
        h, last = ops.gated_scan(d["z"] + sign * s * dirs["z"], d["x"] + sign * s * dirs["x"],
                                 h0=d["h0"] + sign * s * dirs["h0"], reset=d["reset"], form=form)
        return float((h.double() * d["dh"].double()).sum() + (last.double() * d["dh_last"].double()).sum())

    h, _ = ops.gated_scan(d["z"], d["x"], h0=d["h0"], reset=d["reset"], form=form)
    g = ops.gated_scan_backward(d["dh"], d["z"], d["x"], h, h0=d["h0"], reset=d["reset"], dh_last=d["dh_last"],
                                form=form)
    along = sum(float((a.double() * dirs[k].double()).sum()) for a, k in zip(g, ("z", "x", "h0")))
    size = sum(float((a.double() * dirs[k].double()).square().sum()) for a, k in zip(g, ("z", "x", "h0"))) ** 0.5
    assert abs((loss(1) - loss(-1)) / (2 * s) - along) <= 1e-3 * (abs(along) + 10 * size)


def test_another_stream_and_graph_replays(ops):
    """On a side stream, and captured: replays after new inputs give what eager
    calls give."""
    d = data(3000, 1, 64, F32, "sigmoid")
    want = ops.gated_scan(d["z"], d["x"], h0=d["h0"], reset=d["reset"])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    h, last = torch.empty_like(want[0]), torch.empty_like(want[1])
    with torch.cuda.stream(side):
        ops.gated_scan(d["z"], d["x"], h0=d["h0"], reset=d["reset"], out=(h, last))
    side.synchronize()
    assert torch.equal(h, want[0]) and torch.equal(last, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.gated_scan(d["z"], d["x"], h0=d["h0"], reset=d["reset"], out=(h, last))
    for k in range(4):
        d["x"].add_(0.25)
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.gated_scan(d["z"], d["x"], h0=d["h0"], reset=d["reset"])
        assert torch.equal(h, eager[0]) and torch.equal(last, eager[1]), k


def test_growth_inside_a_capture_is_refused():
    from phyz_amd.ops import Ops, OpsError
    fresh = Ops(0)
    z = torch.randn(3000, 1, 64, device="cuda")
    out = (torch.empty_like(z), torch.empty(1, 64, device="cuda"))
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        z.add_(0.0)
        with pytest.raises(OpsError, match="being captured"):
            fresh.gated_scan(z, z, out=out)
    with torch.cuda.stream(side):
        fresh.reserve(1 << 20)
    assert fresh.workspace_bytes >= 1 << 20
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        fresh.gated_scan(z, z, out=out)
    graph.replay()
    torch.cuda.synchronize()
    want = fresh.gated_scan(z, z)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
