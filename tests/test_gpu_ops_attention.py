"""Linear attention on the device against the recurrence in 64 bits, within bounds
that follow from the arithmetic (tests/attend_ref.py)."""
import pytest
import torch

from tests import attend_ref as R

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from phyz_amd.ops import Ops
    return Ops(0)


def inputs(T, B, H, nk, nv, dtype=F32, seed=0, qh=None, kh=None, vh=None, reset=0.03, batch_first=False, slow=3.0):
    g = torch.Generator().manual_seed(seed)
    one = (B, T) if batch_first else (T, B)
    lay = lambda v: v.cuda().transpose(0, 1) if batch_first else v.cuda()  # noqa: E731
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"q": lay(rnd(*one, (qh or H) * nk).to(dtype)), "k": lay(rnd(*one, (kh or H) * nk).to(dtype)),
            "v": lay(rnd(*one, (vh or H) * nv).to(dtype)), "g": lay(torch.nn.functional.logsigmoid(1.5 * rnd(*one, H) + slow)),
            "s0": rnd(B, H, nk, nv).cuda(), "reset": lay(torch.rand(*one, generator=g) < reset) if reset else None,
            "do": lay(rnd(*one, H * nv).to(dtype)), "ds": rnd(B, H, nk, nv).cuda()}


def forward(ops, x, nk, nv, **kw):
    return ops.linear_attention(x["q"], x["k"], x["v"], x["g"], s0=x["s0"], reset=x["reset"], size_k=nk, size_v=nv, **kw)


def backward(ops, x, nk, nv, **kw):
    return ops.linear_attention_backward(x["do"], x["q"], x["k"], x["v"], x["g"], s0=x["s0"], reset=x["reset"], ds=x["ds"],
                                         size_k=nk, size_v=nv, **kw)


def check_forward(got, x, nk, nv, scale=None):
    want, bound = R.attention(x["q"], x["k"], x["v"], x["g"], x["s0"], x["reset"], nk, nv, nk ** -0.5 if scale is None else scale)
    for a, w, b, n in zip(got, want, bound, ("o", "s")):
        R.within(a, w, b, n)


def check_backward(got, x, nk, nv, scale=None):
    want, bound = R.attention_backward(x["do"], x["q"], x["k"], x["v"], x["g"], x["s0"], x["reset"], x["ds"], nk, nv,
                                       nk ** -0.5 if scale is None else scale)
    for a, w, b, n in zip(got, want, bound, ("dq", "dk", "dv", "dg", "ds0")):
        R.within(a, w, b, n)


# steps, worlds, heads, size_k, size_v: one of each, sizes off the tiles (16, 32,
# 64, 128) and on them, steps off the chunks (32 and 64), many chunks and few
# heads (the steps are split), many heads.
SIZES = [(1, 1, 1, 1, 1), (1, 3, 2, 64, 64), (2, 2, 1, 7, 128), (31, 2, 3, 33, 5), (32, 2, 2, 32, 32), (33, 1, 2, 64, 31),
         (63, 2, 1, 65, 64), (64, 3, 2, 64, 64), (65, 2, 2, 128, 33), (100, 1, 2, 128, 128), (129, 2, 1, 16, 100),
         (257, 1, 1, 40, 72), (700, 1, 2, 64, 64), (1100, 1, 1, 128, 64), (20, 150, 3, 12, 20), (70, 300, 4, 8, 16)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T, B, H, nk, nv", SIZES)
def test_forward(ops, T, B, H, nk, nv, dtype):
    x = inputs(T, B, H, nk, nv, dtype, seed=T + nk)
    check_forward(forward(ops, x, nk, nv), x, nk, nv)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T, B, H, nk, nv", SIZES)
def test_backward(ops, T, B, H, nk, nv, dtype):
    x = inputs(T, B, H, nk, nv, dtype, seed=T + nv)
    check_backward(backward(ops, x, nk, nv), x, nk, nv)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("qh, kh, vh", [(1, 1, 6), (6, 2, 2), (3, 6, 1), (2, 1, 3)])
@pytest.mark.parametrize("batch_first", [False, True])
def test_shared_heads(ops, qh, kh, vh, batch_first, dtype):
    x = inputs(90, 3, 6, 24, 40, dtype, 5, qh, kh, vh, batch_first=batch_first)
    check_forward(forward(ops, x, 24, 40, scale=0.7), x, 24, 40, 0.7)
    check_backward(backward(ops, x, 24, 40, scale=0.7), x, 24, 40, 0.7)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B, H, nk, nv, qh, kh, vh", [(1, 1, 1, 1, 1, 1, 1), (3, 4, 64, 64, 4, 4, 4), (2, 6, 33, 5, 1, 2, 3),
                                                      (700, 4, 16, 128, 4, 4, 4), (5, 2, 128, 127, 2, 2, 2),
                                                      (2, 2, 128, 128, 2, 1, 1), (3, 3, 2, 3, 3, 3, 3)])
def test_step(ops, B, H, nk, nv, qh, kh, vh, dtype):
    x = inputs(1, B, H, nk, nv, dtype, 3, qh, kh, vh, reset=0.3)
    s = x["s0"].clone()
    o = ops.linear_attention_step(x["q"][0], x["k"][0], x["v"][0], x["g"][0], s, reset=x["reset"][0], size_k=nk, size_v=nv)
    check_forward((o[None], s), x, nk, nv)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_steps_are_the_scan(ops, dtype):
    """States differ by the order of f32 sums, outputs by that and one rounding: both
    are within their bounds of the same recurrence."""
    x = inputs(70, 4, 3, 32, 48, dtype, 8)
    s, outs = x["s0"].clone(), []
    for t in range(70):
        outs.append(ops.linear_attention_step(x["q"][t], x["k"][t], x["v"][t], x["g"][t], s, reset=x["reset"][t]))
    check_forward((torch.stack(outs), s), x, 32, 48)


@pytest.mark.parametrize("T, B, H", [(150, 2, 2), (1500, 1, 1)])
def test_gates_of_all_sizes(ops, T, B, H):
    """Gates that keep everything, that forget at once, and in between; where g is
    below -104 or a reset is set, nothing of before is left."""
    x = inputs(T, B, H, 32, 64, F32, 6, reset=0.01)
    gen = torch.Generator().manual_seed(1)
    pick = torch.randint(0, 6, x["g"].shape, generator=gen).cuda()
    for i, v in enumerate((0.0, -1e-6, -0.3, -20.0, -103.0, -float("inf"))):
        x["g"][pick == i] = v
    check_forward(forward(ops, x, 32, 64), x, 32, 64)
    check_backward(backward(ops, x, 32, 64), x, 32, 64)


def test_gates_that_keep(ops):
    """g = 0 all through: sums over all steps."""
    x = inputs(900, 1, 2, 64, 32, F32, 7, reset=0)
    x["g"].zero_()
    check_forward(forward(ops, x, 64, 32), x, 64, 32)
    check_backward(backward(ops, x, 64, 32), x, 64, 32)


def test_gates_that_grow(ops):
    """g above 0, as far as its documentation goes: up to 2^32 in 16 steps, against
    the bound's own growth."""
    x = inputs(48, 2, 2, 16, 16, F32, 9, reset=0)
    x["g"].uniform_(0.0, 1.2)
    check_forward(forward(ops, x, 16, 16), x, 16, 16)


def test_one_gate_a_head(ops):
    x = inputs(80, 3, 4, 32, 32, BF16, 10)
    rates = torch.tensor([-0.5, -0.1, -0.01, 0.0], device="cuda")
    x["g"] = rates.expand(80, 3, 4)
    o, s = ops.linear_attention(x["q"], x["k"], x["v"], rates, s0=x["s0"], reset=x["reset"])
    check_forward((o, s), x, 32, 32)
    check_backward(ops.linear_attention_backward(x["do"], x["q"], x["k"], x["v"], rates, s0=x["s0"], reset=x["reset"],
                                                 ds=x["ds"]), x, 32, 32)
    state = x["s0"].clone()
    a = ops.linear_attention_step(x["q"][0], x["k"][0], x["v"][0], rates, state, reset=x["reset"][0])
    assert a.shape == (3, 128)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T, bad", [(150, 40), (150, 64), (40, 0), (1500, 700)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_what_is_not_finite_stays_in_its_episode(ops, T, bad, value, dtype):
    """An episode of one head diverges and ends; steps before, the next episode and
    the other heads are as if it had not."""
    x = inputs(T, 2, 2, 32, 32, dtype, 11, reset=0)
    x["reset"] = torch.zeros(T, 2, dtype=torch.bool, device="cuda")
    x["reset"][bad + 10] = True
    want, wb = R.attention(x["q"], x["k"], x["v"], x["g"], x["s0"], x["reset"], 32, 32, 32 ** -0.5)
    grads, gb = R.attention_backward(x["do"], x["q"], x["k"], x["v"], x["g"], x["s0"], x["reset"], x["ds"], 32, 32, 32 ** -0.5)
    for name, at in (("k", (bad, 0, 5)), ("v", (bad, 0, 7)), ("q", (bad, 0, 3)), ("g", (bad, 0, 0))):
        y = dict(x)
        y[name] = x[name].clone()
        y[name][at] = value
        o, s = forward(ops, y, 32, 32)
        clean = torch.ones(T, 2, 64, dtype=torch.bool)
        clean[bad:bad + 10, 0, :32] = False
        got = torch.where(clean, o.cpu().double(), want[0])
        R.within(got, want[0], wb[0], f"{name}: o")
        R.within(s, want[1], wb[1], f"{name}: s")
        assert not torch.isfinite(o[bad, 0, :32]).all(), name
        dq, dk, dv, dg, ds0 = backward(ops, y, 32, 32)
        for got, w, b, what in ((dq, grads[0], gb[0], "dq"), (dk, grads[1], gb[1], "dk"), (dv, grads[2], gb[2], "dv")):
            # Another world, another head, and the episode behind.
            for part in ((slice(None), 1), (slice(None), 0, slice(32, 64)), (slice(bad + 10, None), 0)):
                R.within(got[part], w[part], b[part], f"{name}: {what}")
        R.within(dg[:, 1], grads[3][:, 1], gb[3][:, 1], f"{name}: dg")
        R.within(ds0[1], grads[4][1], gb[4][1], f"{name}: ds0")


def test_a_first_state_that_is_not_finite(ops):
    x = inputs(100, 2, 2, 16, 16, F32, 12, reset=0)
    x["reset"] = torch.zeros(100, 2, dtype=torch.bool, device="cuda")
    x["reset"][3] = True
    want, bound = R.attention(x["q"], x["k"], x["v"], x["g"], x["s0"], x["reset"], 16, 16, 0.25)
    x["s0"] = torch.full_like(x["s0"], float("nan"))
    o, s = forward(ops, x, 16, 16)
    R.within(o[3:], want[0][3:], bound[0][3:], "o")
    R.within(s, want[1], bound[1], "s")
    s = x["s0"].clone()
    x["reset"][0] = True
    o = ops.linear_attention_step(x["q"][0], x["k"][0], x["v"][0], x["g"][0], s, reset=x["reset"][0])
    assert torch.isfinite(o).all() and torch.isfinite(s).all()


def test_without_optional_tensors(ops):
    x = inputs(70, 2, 2, 32, 32, F32, 13, reset=0)
    q, k, v, g = x["q"], x["k"], x["v"], x["g"]
    x["s0"], x["ds"] = None, None
    check_forward(ops.linear_attention(q, k, v, g), x, 32, 32)
    o, last = torch.empty_like(v), None
    ops.linear_attention(q, k, v, g, out=(o, None))
    assert torch.equal(o, ops.linear_attention(q, k, v, g)[0])
    want, bound = R.attention_backward(x["do"], q, k, v, g, None, None, None, 32, 32, 32 ** -0.5)
    got = ops.linear_attention_backward(x["do"], q, k, v, g, need_dg=False)
    assert got[3] is None
    for i in (0, 1, 2, 4):
        R.within(got[i], want[i], bound[i], str(i))


def test_no_steps_and_no_worlds(ops):
    x = inputs(4, 2, 3, 8, 16, F32, 14)
    cut = {n: (t[:0] if n in ("q", "k", "v", "g", "reset", "do") else t) for n, t in x.items()}
    o, s = forward(ops, cut, 8, 16)
    assert o.shape == (0, 2, 48) and torch.equal(s, x["s0"])
    cut["s0"] = None
    assert not forward(ops, cut, 8, 16)[1].any()
    ds0 = backward(ops, cut, 8, 16)[4]
    assert torch.equal(ds0, x["ds"])
    none = {n: (t[:, :0] if n in ("q", "k", "v", "g", "reset", "do") else t[:0]) for n, t in x.items()}
    assert forward(ops, none, 8, 16)[0].shape == (4, 0, 48)
    backward(ops, none, 8, 16)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_views_and_their_surroundings(ops, dtype):
    """q, k and v as slices of one buffer's rows at odd offsets, outputs as slices of
    others: the same results, nothing beside them written."""
    T, B, H, nk, nv = 75, 3, 2, 24, 40
    x = inputs(T, B, H, nk, nv, dtype, 15)
    plain, grads = forward(ops, x, nk, nv), backward(ops, x, nk, nv)
    wide = torch.full((T, B, 3 + 2 * H * nk + H * nv + 2), 9.0, dtype=dtype, device="cuda")
    cuts = {"q": slice(3, 3 + H * nk), "k": slice(3 + H * nk, 3 + 2 * H * nk), "v": slice(3 + 2 * H * nk, 3 + 2 * H * nk + H * nv)}
    y = dict(x)
    for n, c in cuts.items():
        wide[..., c] = x[n]
        y[n] = wide[..., c]
    y["g"] = torch.stack([x["g"], x["g"] + 1], -1)[..., 0]
    states = torch.full((B, H + 1, nk * nv + 3), 9.0, device="cuda")
    last = states[:, :H, :nk * nv].view(B, H, nk, nv) if False else states.as_strided((B, H, nk, nv), ((H + 1) * (nk * nv + 3), nk * nv + 3, nv, 1))
    obuf = torch.full((T, B, H * nv + 5), 9.0, dtype=dtype, device="cuda")
    o, s = forward(ops, y, nk, nv, out=(obuf[..., 1:1 + H * nv], last))
    assert torch.equal(o, plain[0]) and torch.equal(s, plain[1])
    assert bool((obuf[..., 0] == 9).all()) and bool((obuf[..., 1 + H * nv:] == 9).all())
    assert bool((states[:, H] == 9).all()) and bool((states[..., nk * nv:] == 9).all())
    dw = torch.full_like(wide, 9.0)
    dgs = torch.full((T, B, H, 2), 9.0, device="cuda")
    got = backward(ops, y, nk, nv, out=(dw[..., cuts["q"]], dw[..., cuts["k"]], dw[..., cuts["v"]], dgs[..., 1], torch.empty_like(x["s0"])))
    for a, b in zip(got, grads):
        assert torch.equal(a, b)
    assert bool((dw[..., :3] == 9).all()) and bool((dw[..., -2:] == 9).all()) and bool((dgs[..., 0] == 9).all())


def test_repeats_bit_for_bit(ops):
    for T, B, H in ((300, 2, 3), (2500, 1, 1)):
        x = inputs(T, B, H, 64, 64, BF16, 16, qh=1, kh=1)
        a, b = forward(ops, x, 64, 64), backward(ops, x, 64, 64)
        for _ in range(3):
            assert all(torch.equal(u, w) for u, w in zip(a, forward(ops, x, 64, 64)))
            assert all(torch.equal(u, w) for u, w in zip(b, backward(ops, x, 64, 64)))


def test_gradients_against_differences(ops):
    """Each input's gradient along a random direction against the loss's central
    difference, in f32: steps of 1e-2 of unit directions leave (1e-2)^2 of third
    derivatives and 2^-24 of the loss's terms over 1e-2; 3e-3 of the norm covers both."""
    x = inputs(50, 2, 2, 16, 24, F32, 17)
    gen = torch.Generator().manual_seed(18)

    def loss():
        o, s = forward(ops, x, 16, 24)
        return float((o.double() * x["do"].double()).sum() + (s.double() * x["ds"].double()).sum())

    grads = dict(zip(("q", "k", "v", "g", "s0"), backward(ops, x, 16, 24)))
    for n, grad in grads.items():
        d = torch.randn(x[n].shape, generator=gen).cuda()
        d /= d.norm()
        keep, h = x[n], 1e-2
        x[n] = keep + h * d
        up = loss()
        x[n] = keep - h * d
        down = loss()
        x[n] = keep
        assert abs((up - down) / (2 * h) - float((grad.double() * d.double()).sum())) <= 3e-3 * float(grad.double().norm()), n


def test_another_stream_and_graphs(ops):
    """On a side stream, and captured with the backward pass, replayed between eager
    calls."""
    x = inputs(2100, 1, 2, 64, 64, BF16, 19, kh=1)
    want, grads = forward(ops, x, 64, 64), backward(ops, x, 64, 64)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a, b = forward(ops, x, 64, 64), backward(ops, x, 64, 64)
    side.synchronize()
    assert all(torch.equal(u, w) for u, w in zip((*want, *grads), (*a, *b)))
    outs, gouts = tuple(torch.empty_like(t) for t in want), tuple(torch.empty_like(t) for t in grads)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        forward(ops, x, 64, 64, out=outs)
        backward(ops, x, 64, 64, out=gouts)
    for _ in range(3):
        for t in (*outs, *gouts):
            t.fill_(7.0)
        graph.replay()
        other = forward(ops, x, 64, 64)
        torch.cuda.synchronize()
        assert all(torch.equal(u, w) for u, w in zip((*want, *grads), (*outs, *gouts)))
        assert torch.equal(other[0], want[0])


def test_rows_past_two_gigabytes(ops):
    """Strides that put the last steps 2^31 elements behind the first."""
    T, B, H, n = 70, 2, 1, 32
    x = inputs(T, B, H, n, n, BF16, 20)
    plain = forward(ops, x, n, n)
    step = (1 << 31) // (T - 6)
    big = torch.empty(step * (T - 1) + B * n + 1, dtype=BF16, device="cuda")
    far = big.as_strided((T, B, n), (step, n, 1))
    far.copy_(x["v"])
    y = dict(x, v=far)
    got = forward(ops, y, n, n)
    assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
    dv = far
    want = backward(ops, x, n, n)
    got = backward(ops, x, n, n, out=(*(torch.empty_like(t) for t in want[:2]), dv, *(torch.empty_like(t) for t in want[3:])))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
