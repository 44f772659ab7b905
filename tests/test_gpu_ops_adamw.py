"""AdamW over lists of tensors on the device against 64 bits; moments of 8 bits
code by code."""
import math

import numpy as np
import pytest
import torch

from tests import attend_ref as R

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
HYPER = {"lr": 3e-3, "betas": (0.9, 0.99), "eps": 1e-8, "weight_decay": 0.1}
# One element, off and on the 4 of a lane, the 256 of a wave and the 4096 of a
# workgroup, no elements, several axes.
SHAPES = [(1,), (3,), (4, 1), (5, 51), (256,), (257,), (0,), (64, 64), (4097,), (3, 5, 7, 2), (1000, 37), ()]


@pytest.fixture(scope="module")
def ops():
    from phyz_amd.ops import Ops
    return Ops(0)


def tensors(shapes, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(s, generator=g) * torch.exp(torch.randn((), generator=g))).to(dtype).cuda() for s in shapes]


@pytest.mark.parametrize("w_type", [F32, BF16], ids=["w f32", "w bf16"])
@pytest.mark.parametrize("g_type", [F32, BF16], ids=["g f32", "g bf16"])
def test_steps(ops, w_type, g_type):
    w = tensors(SHAPES, w_type, 1)
    m, v, e, step = ops.adamw_state(w)
    assert e is None
    for t in range(1, 4):
        g = tensors(SHAPES, g_type, 10 + t, 1e-2)
        before = [[x.clone() for x in l] for l in (w, m, v)]
        ops.adamw_step(w, g, m, v, step, **HYPER)
        assert int(step) == t
        for i in range(len(w)):
            want, bound = R.adamw(before[0][i], g[i], before[1][i], before[2][i], t, *HYPER.values())
            for got, a, b, n in zip((w[i], m[i], v[i]), want, bound, "wmv"):
                R.within(got, a, b, f"{n}[{i}]")


def test_many_tensors_of_both_types(ops):
    """More tensors than a launch holds, types mixed."""
    shapes = [(1 + (37 * i) % 700,) for i in range(200)]
    w = [t.to(F32 if i % 3 else BF16) for i, t in enumerate(tensors(shapes, F32, 2))]
    g = [t.to(F32 if i % 2 else BF16) for i, t in enumerate(tensors(shapes, F32, 3, 1e-3))]
    m, v, _, step = ops.adamw_state(w)
    start = [x.clone() for x in w]
    step.fill_(999)
    ops.adamw_step(w, g, m, v, step, **HYPER)
    for i in range(200):
        want, bound = R.adamw(start[i], g[i], torch.zeros(shapes[i]), torch.zeros(shapes[i]), 1000, *HYPER.values())
        for got, a, b, n in zip((w[i], m[i], v[i]), want, bound, "wmv"):
            R.within(got, a, b, f"{n}[{i}]")


def numbers(n, seed):
    """f32 values over f32's range and within blocks, zeros among them."""
    r = np.random.RandomState(seed)
    x = r.standard_normal(n).astype(np.float32) * np.exp2(r.uniform(-22, 0, n)).astype(np.float32)
    x[r.rand(n) < 0.05] = 0
    x *= np.exp2(np.repeat(r.uniform(-30, 10, -(-n // 256)), 256)[:n]).astype(np.float32)
    return x


@pytest.mark.parametrize("seed, t", [(0, 1), (12345, 7), (2 ** 32 - 1, 70000)])
def test_codes(ops, seed, t):
    """Every code and exponent, against a search through what the codes stand for.
    With betas of 0 the moments are g and g^2."""
    sizes = [1, 255, 256, 700]
    g = [torch.from_numpy(numbers(n, n + seed % 1000)).cuda() for n in sizes]
    g[3][300:520] = 0
    w = [torch.zeros_like(x) for x in g]
    m, v, e, step = ops.adamw_state(w, bits=8)
    step.fill_(t - 1)
    ops.adamw_step(w, g, m, v, step, exponents=e, betas=(0.0, 0.0), seed=seed)
    mv, vv = ops.adamw_values(m, v, e)
    for k, n in enumerate(sizes):
        for x, codes, values, top, signed, row, which in (
                (g[k].cpu().numpy(), m[k], mv[k], 14, True, 0, 0),
                ((g[k].cpu().numpy() * g[k].cpu().numpy()), v[k], vv[k], 30, False, 1, 1)):
            codes, ex = codes.cpu().tolist(), e[k][row].cpu().tolist()
            values = values.double().cpu().tolist()
            for blk in range(-(-n // 256)):
                part = x[blk * 256:(blk + 1) * 256]
                most = float(np.abs(part).max())
                want = max(40, math.frexp(most)[1] + 126) if most else 40
                assert ex[blk] == want
                table = R.code_values(want, top, signed)
                for i, y in enumerate(part):
                    at = blk * 256 + i
                    c = R.encode(float(y), want, top, signed, R.dither(seed, t, k, at)[which])
                    assert codes[at] == c, (k, at, float(y), codes[at], c)
                    assert values[at] == table[c]


def test_eight_bits_follow_32(ops):
    """w goes by the moments before they are rounded: one step from decoded moments
    is the 32-bit step, bit for bit."""
    shapes = [(300, 7), (5,), (4096, 2)]
    w = tensors(shapes, F32, 4)
    m, v, e, step = ops.adamw_state(w, bits=8)
    for k in range(3):
        g = tensors(shapes, BF16, 20 + k, 1e-3)
        mv, vv = ops.adamw_values(m, v, e)
        w32, m32, v32, step32 = [x.clone() for x in w], [x.float() for x in mv], [x.float() for x in vv], step.clone()
        ops.adamw_step(w32, g, m32, v32, step32, **HYPER)
        ops.adamw_step(w, g, m, v, step, exponents=e, seed=5, **HYPER)
        assert torch.equal(step, step32)
        for a, b in zip(w, w32):
            assert torch.equal(a, b)
        # Codes are off by less than one step of theirs: 1/8 of the value.
        for got, exact in zip((*ops.adamw_values(m, v, e)[0], *ops.adamw_values(m, v, e)[1]), (*m32, *v32)):
            tiny = exact.abs().max() * 2.0 ** -15
            assert bool(((got.float() - exact).abs() <= exact.abs() / 8 + tiny).all())


def test_rounding_is_right_on_average(ops):
    """v's moving average with 0.999 rises by a thousandth a step, far less than a
    code: over 400 steps its mean over 65536 elements is off by their random walk
    alone, 0.07 sqrt(400) / sqrt(65536) of it at most (a step's deviation is below
    half a code's width, 1/16, with a chance below 1/8)."""
    n = 65536
    w, g = [torch.zeros(n, device="cuda")], [torch.full((n,), 1e-2, device="cuda")]
    m, v, e, step = ops.adamw_state(w, bits=8)
    for _ in range(400):
        ops.adamw_step(w, g, m, v, step, exponents=e, betas=(0.9, 0.999))
    want = 1e-4 * (1 - 0.999 ** 400)
    got = float(ops.adamw_values(m, v, e)[1][0].double().mean())
    assert abs(got / want - 1) < 0.01
    assert abs(float(ops.adamw_values(m, v, e)[0][0].double().mean()) / 1e-2 - 1) < 0.01


def test_what_is_not_finite(ops):
    """Beside infinities and NaN, a block's other elements are as without them; a
    gradient of 0 leaves moments of 0, and v's small values do not vanish."""
    g = [torch.randn(600, generator=torch.Generator().manual_seed(1)).cuda() * 1e-3]
    bad = [g[0].clone()]
    bad[0][5], bad[0][300], bad[0][301] = float("nan"), float("inf"), -float("inf")
    out = []
    for x in (g, bad):
        w = [torch.ones(600, device="cuda")]
        m, v, e, step = ops.adamw_state(w, bits=8)
        ops.adamw_step(w, x, m, v, step, exponents=e)
        mv, vv = ops.adamw_values(m, v, e)
        out.append((w[0], mv[0], vv[0]))
    fine = torch.ones(600, dtype=torch.bool, device="cuda")
    fine[[5, 300, 301]] = False
    for a, b in zip(*out):
        assert torch.equal(a[fine], b[fine])
        assert not torch.isfinite(b[5])
    assert torch.isnan(out[1][1][~fine]).all() and torch.isnan(out[1][2][~fine]).all()
    w, g = [torch.ones(4, device="cuda")], [torch.tensor([1.0, 0.0, 1e-12, 1e-4], device="cuda")]
    m, v, e, step = ops.adamw_state(w, bits=8)
    ops.adamw_step(w, g, m, v, step, exponents=e, betas=(0.9, 0.999))
    vv = ops.adamw_values(m, v, e)[1][0]
    assert float(vv[1]) == 0 and float(vv[2]) > 0 and torch.isfinite(w[0]).all()


def test_replays_count_on(ops):
    """A captured step replayed is the next step: the count, the bias corrections and
    the random bits go on, as eager steps do."""
    for bits in (32, 8):
        def start():
            w = tensors([(500,), (33, 40)], F32, 6)
            return w, ops.adamw_state(w, bits=bits)
        g = tensors([(500,), (33, 40)], F32, 7, 1e-3)
        we, (me, ve, ee, se) = start()
        for _ in range(4):
            ops.adamw_step(we, g, me, ve, se, exponents=ee, seed=3, **HYPER)
        w, (m, v, e, step) = start()
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            ops.adamw_step(w, g, m, v, step, exponents=e, seed=3, **HYPER)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.adamw_step(w, g, m, v, step, exponents=e, seed=3, **HYPER)
        for _ in range(3):
            graph.replay()
            ops.adamw_step(*[[torch.ones(9, device="cuda")] for _ in range(4)], torch.zeros(1, dtype=torch.int64, device="cuda"))
            torch.cuda.synchronize()
        assert int(step) == 4
        for a, b in zip((*w, *m, *v, *(e or [])), (*we, *me, *ve, *(ee or []))):
            assert torch.equal(a, b)


def test_odd_addresses(ops):
    """Tensors that begin anywhere in a buffer, and what stands between them."""
    sizes, at, places = [3, 257, 1000, 4099, 1], 1, []
    for n in sizes:
        places.append(slice(at, at + n))
        at += n + 1
    buf = {k: torch.full((at,), 7.0, device="cuda") for k in "wgmv"}
    code = {k: torch.full((at,), 7, dtype=torch.uint8, device="cuda") for k in "mv"}
    for bits in (32, 8):
        w, g = tensors([(n,) for n in sizes], F32, 8), tensors([(n,) for n in sizes], F32, 9, 1e-2)
        m, v, e, step = ops.adamw_state(w, bits=bits)
        src = buf if bits == 32 else {**buf, **code}
        cut = {k: [src[k][p] for p in places] for k in "wgmv"}
        for k, l in zip("wgmv", (w, g, m, v)):
            for a, b in zip(cut[k], l):
                a.copy_(b)
        e2, step2 = None if e is None else [x.clone() for x in e], step.clone()
        for _ in range(2):
            ops.adamw_step(w, g, m, v, step, exponents=e, **HYPER)
            ops.adamw_step(cut["w"], cut["g"], cut["m"], cut["v"], step2, exponents=e2, **HYPER)
        for k, l in zip("wmv", (w, m, v)):
            for a, b in zip(cut[k], l):
                assert torch.equal(a, b)
        gaps = torch.ones(at, dtype=torch.bool, device="cuda")
        for p in places:
            gaps[p] = False
        for t in src.values():
            assert bool((t[gaps] == 7).all())
