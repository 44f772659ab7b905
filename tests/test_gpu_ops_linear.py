"""The linear layer, its epilogue and its gradients on the device against 64
bits, element by element within bounds of their arithmetic (tests/ops_ref.py)."""
import pytest
import torch

from tests import ops_ref as R

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
ACTS = ["none", "tanh", "relu", "silu", "gelu"]
#: rows, n_in, n_out: single rows and columns, the policy's observation widths,
#: sizes on and off every tile, few rows through wide layers, long sums.
SHAPES = [(1, 1, 1), (1, 64, 64), (1, 2048, 515), (2, 55, 256), (3, 7, 5), (8, 1024, 1000), (16, 512, 2048),
          (17, 300, 129), (33, 67, 31), (64, 64, 64), (100, 129, 65), (127, 256, 257), (128, 128, 128), (130, 1000, 1),
          (300, 1, 70), (511, 96, 384), (1025, 55, 256), (2048, 520, 264), (4096, 256, 8), (777, 1001, 333)]


@pytest.fixture(scope="module")
def ops():
    from phyz_amd.ops import Ops
    return Ops(0)


def data(m, k, n, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)

    def r(*s, scale=1.0):
        return (torch.randn(*s, generator=g) * scale).to("cuda", dtype)

    return {"x": r(m, k), "w": r(n, k, scale=k ** -0.5), "bias": r(n), "residual": r(m, n), "dy": r(m, n),
            "pre": r(m, n, scale=2.0)}


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(ops, shape, dtype):
    d = data(*shape, dtype)
    act = ACTS[sum(shape) % 5]
    bias = d["bias"] if sum(shape) % 3 else None
    residual = d["residual"] if sum(shape) % 2 else None
    y, pre = ops.linear(d["x"], d["w"], bias=bias, act=act, residual=residual, save_pre=True)
    wy, wp, by, bp = R.linear(d["x"], d["w"], bias, residual, act, dtype)
    R.within(y, wy, by, "y")
    R.within(pre, wp, bp, "pre")
    assert torch.equal(y, ops.linear(d["x"], d["w"], bias=bias, act=act, residual=residual))
    got = ops.linear_backward(d["dy"], d["x"], d["w"], pre=d["pre"] if act != "none" else None, act=act)
    want, bounds = R.linear_backward(d["dy"], d["x"], d["w"], d["pre"] if act != "none" else None, act, dtype)
    for name, a, b, c in zip(("dx", "dw", "db"), got, want, bounds):
        R.within(a, b, c, name)


#: Few tiles and a long contraction, in one product or another, at sizes off the
#: vector; and rows about where another kernel or another split of rows begins.
LONG = [(2, 57, 914), (125, 1618, 2), (357, 1647, 67), (2149, 45, 1003), (40, 3001, 9), (33, 520, 300), (48, 2048, 515),
        (64, 1000, 72), (65, 1000, 72), (512, 40, 33), (513, 40, 33), (511, 24, 700), (128, 40, 33), (129, 40, 33)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", LONG, ids=str)
def test_long_contractions(ops, shape, dtype):
    test_forward_and_backward(ops, shape, dtype)


#: Large enough for every tile, for split contractions and for operands that
#: are copied first, on and off the tiles' sizes.
LARGE = [(4096, 4096, 64, "silu"), (3001, 1024, 2056, "none"), (257, 4104, 520, "tanh"), (9000, 131, 1003, "gelu"),
         (70000, 64, 72, "relu"), (2100, 1001, 2049, "none")]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", LARGE, ids=str)
def test_large(ops, shape, dtype):
    m, k, n, act = shape
    d = data(m, k, n, dtype, seed=4)
    y, pre = ops.linear(d["x"], d["w"], bias=d["bias"], act=act, residual=d["residual"], save_pre=True)
    wy, wp, by, bp = R.linear(d["x"], d["w"], d["bias"], d["residual"], act, dtype)
    R.within(y, wy, by, "y")
    R.within(pre, wp, bp, "pre")
    p = d["pre"] if act != "none" else None
    got = ops.linear_backward(d["dy"], d["x"], d["w"], pre=p, act=act)
    want, bounds = R.linear_backward(d["dy"], d["x"], d["w"], p, act, dtype)
    for name, a, b, c in zip(("dx", "dw", "db"), got, want, bounds):
        R.within(a, b, c, name)
    for a, b in zip(got, ops.linear_backward(d["dy"], d["x"], d["w"], pre=p, act=act)):
        assert torch.equal(a, b)


def test_rows_far_apart(ops):
    """Rows 32 MiB apart: a tile's rows leave 32-bit offsets."""
    m, k, n = 300, 64, 48
    big = torch.zeros((m - 1) * (1 << 24) + k, dtype=BF16, device="cuda")
    x = torch.as_strided(big, (m, k), (1 << 24, 1))
    x.copy_(torch.randn(m, k, device="cuda"))
    w = torch.randn(n, k, device="cuda").to(BF16)
    assert torch.equal(ops.linear(x, w), ops.linear(x.contiguous(), w))
    dy = torch.randn(m, n, device="cuda").to(BF16)
    for a, b in zip(ops.linear_backward(dy, x, w), ops.linear_backward(dy, x.contiguous(), w)):
        assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-2)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("act", ACTS)
def test_activations(ops, act, dtype):
    d = data(70, 40, 90, dtype, seed=1)
    d["x"] *= 4
    y, pre = ops.linear(d["x"], d["w"], bias=d["bias"], act=act, residual=d["residual"], save_pre=True)
    wy, wp, by, bp = R.linear(d["x"], d["w"], d["bias"], d["residual"], act, dtype)
    R.within(y, wy, by, "y")
    got = ops.linear_backward(d["dy"], d["x"], d["w"], pre=pre, act=act)
    want, bounds = R.linear_backward(d["dy"], d["x"], d["w"], pre, act, dtype)
    for name, a, b, c in zip(("dx", "dw", "db"), got, want, bounds):
        R.within(a, b, c, name)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(4, 96, 200), (20, 64, 72), (300, 200, 264), (600, 1024, 512)], ids=str)
def test_strided_views(ops, shape, dtype):
    """Rows inside wider rows, at offsets of one element, leave the rest alone."""
    m, k, n = shape
    d = data(*shape, dtype)

    def inside(t, at):
        wide = torch.full((t.shape[0], t.shape[1] + 9), 3.0, dtype=dtype, device="cuda")
        v = wide[:, at:at + t.shape[1]]
        v.copy_(t)
        return wide, v

    _, x = inside(d["x"], 1)
    _, w = inside(d["w"], 3)
    _, res = inside(d["residual"], 5)
    wide, y = inside(torch.zeros_like(d["residual"]), 7)
    bias = torch.stack([d["bias"], d["bias"]], 1)[:, 0]
    ops.linear(x, w, bias=bias, act="silu", residual=res, out=y)
    assert torch.equal(y, ops.linear(d["x"], d["w"], bias=d["bias"], act="silu", residual=d["residual"]))
    y.fill_(3.0)
    assert (wide == 3).all()
    _, dy = inside(d["dy"], 1)
    _, pre = inside(d["pre"], 2)
    for a, b in zip(ops.linear_backward(dy, x, w, pre=pre, act="gelu"),
                    ops.linear_backward(d["dy"], d["x"], d["w"], pre=d["pre"], act="gelu")):
        assert torch.equal(a, b)


def test_residual_in_place_and_batched_shapes(ops):
    d = data(24, 32, 32, F32)
    want = ops.linear(d["x"], d["w"], residual=d["residual"])
    y = d["residual"].clone()
    assert ops.linear(d["x"], d["w"], residual=y, out=y) is y
    assert torch.equal(y, want)
    y3 = ops.linear(d["x"].view(2, 3, 4, 32), d["w"], residual=d["residual"].view(2, 3, 4, 32))
    assert y3.shape == (2, 3, 4, 32) and torch.equal(y3.view(24, 32), want)
    dx, dw, db = ops.linear_backward(d["dy"].view(2, 12, 32), d["x"].view(2, 12, 32), d["w"])
    flat = ops.linear_backward(d["dy"], d["x"], d["w"])
    assert dx.shape == (2, 12, 32) and torch.equal(dx.view(24, 32), flat[0]) and torch.equal(dw, flat[1])


def test_broadcast_rows(ops):
    """One row of inputs (and of output gradients) for all: stride 0."""
    d = data(50, 24, 40, F32)
    x, dy = d["x"][:1].expand(50, 24), d["dy"][:1].expand(50, 40)
    assert torch.equal(ops.linear(x, d["w"]), ops.linear(x.contiguous(), d["w"]))
    for a, b in zip(ops.linear_backward(dy, x, d["w"]), ops.linear_backward(dy.contiguous(), x.contiguous(), d["w"])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_partial_gradients_and_empty(ops, dtype):
    d = data(40, 24, 56, dtype)
    full = ops.linear_backward(d["dy"], d["x"], d["w"], pre=d["pre"], act="tanh")
    for k in range(3):
        need = [i == k for i in range(3)]
        got = ops.linear_backward(d["dy"], d["x"], d["w"], pre=d["pre"], act="tanh", need_dx=need[0], need_dw=need[1],
                                  need_db=need[2])
        assert torch.equal(got[k], full[k]) and all(got[i] is None for i in range(3) if i != k)
    x0, w = d["x"][:0], d["w"]
    assert ops.linear(x0, w).shape == (0, 56)
    dx, dw, db = ops.linear_backward(d["dy"][:0], x0, w)
    assert dx.shape == (0, 24) and not dw.any() and not db.any()
    # No inputs: the bias alone. No outputs: no gradient.
    y = ops.linear(d["x"][:, :0], w[:, :0], bias=d["bias"], act="relu", residual=d["residual"])
    want = (torch.relu(d["bias"].float())[None] + d["residual"].float()).to(dtype)
    assert torch.equal(y, want)
    dx, dw, db = ops.linear_backward(d["dy"][:, :0], d["x"], w[:0])
    assert not dx.any() and dw.shape == (0, 24) and db.shape == (0,)


@pytest.mark.parametrize("rows", [5, 200])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_infinite_and_nan_inputs(ops, dtype, rows):
    """One infinite or NaN input reaches its own row alone, as products in f32
    have it: infinite where its weight is not 0."""
    d = data(rows, 48, 70, dtype)
    clean = ops.linear(d["x"], d["w"])
    d["x"][1, 3], d["x"][3, 5] = float("inf"), float("nan")
    d["w"][9, 3] = 0.0
    y = ops.linear(d["x"], d["w"])
    keep = [i for i in range(rows) if i not in (1, 3)]
    same = [j for j in range(70) if j != 9]
    assert torch.equal(y[keep][:, same], clean[keep][:, same])
    assert torch.isnan(y[3]).all() and torch.isnan(y[1, 9])
    sign = torch.sign(d["w"][same, 3].float()) * float("inf")
    assert torch.equal(y[1, same].float(), sign)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_infinite_inputs_of_large_products(ops, dtype):
    """The same through the large products, forward and backward, split sums too."""
    m, k, n = 2000, 520, 1032
    d = data(m, k, n, dtype)
    clean = ops.linear(d["x"], d["w"])
    dxc, dwc, _ = ops.linear_backward(d["dy"], d["x"], d["w"])
    x, dy = d["x"].clone(), d["dy"].clone()
    x[7, 3], dy[1500, 9] = float("inf"), float("-inf")
    y = ops.linear(x, d["w"])
    assert torch.equal(y[7].float(), torch.sign(d["w"][:, 3].float()) * float("inf"))
    y[7] = clean[7]
    assert torch.equal(y, clean)
    dx, dw, _ = ops.linear_backward(dy, d["x"], d["w"])
    assert torch.equal(dx[1500].float(), torch.sign(d["w"][9].float()) * float("-inf"))
    assert torch.equal(dw[9].float(), torch.sign(d["x"][1500].float()) * float("-inf"))
    dx[1500], dw[9] = dxc[1500], dwc[9]
    assert torch.equal(dx, dxc) and torch.equal(dw, dwc)


def test_f32_in_pieces(ops):
    """Large enough to be cut into bf16 pieces: within the bounds of f32, and an
    infinite input reaches its own row alone, with its sign."""
    m, k, n = 4100, 2056, 1032
    d = data(m, k, n, F32, seed=8)
    y = ops.linear(d["x"], d["w"], bias=d["bias"], act="silu")
    wy, _, by, _ = R.linear(d["x"], d["w"], d["bias"], None, "silu", F32)
    R.within(y, wy, by, "y")
    got = ops.linear_backward(d["dy"], d["x"], d["w"], pre=d["pre"], act="gelu")
    want, bounds = R.linear_backward(d["dy"], d["x"], d["w"], d["pre"], "gelu", F32)
    for name, a, b, c in zip(("dx", "dw", "db"), got, want, bounds):
        R.within(a, b, c, name)
    plain = ops.linear(d["x"], d["w"])
    x = d["x"].clone()
    x[17, 2000] = float("-inf")
    x[4099, 1] = float("nan")
    y = ops.linear(x, d["w"])
    assert torch.equal(y[17], torch.sign(d["w"][:, 2000]) * float("-inf")) and torch.isnan(y[4099]).all()
    y[17], y[4099] = plain[17], plain[4099]
    assert torch.equal(y, plain)


def test_wide_range_in_f32(ops):
    """f32 operands keep their range and all 24 bits: magnitudes from 2^-60 to
    2^60 in one product."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(64, 128, generator=g) * torch.exp2(torch.randint(-60, 60, (64, 128), generator=g).float())
    w = torch.randn(80, 128, generator=g)
    y = ops.linear(x.cuda(), w.cuda())
    want, _, bound, _ = R.linear(x, w, None, None, "none", F32)
    R.within(y, want, bound, "y")


@pytest.mark.parametrize("act", ACTS)
def test_gradient_against_differences(ops, act):
    """The central difference of the loss along a direction against the
    gradients' inner product with it; 2e-3 covers the step's third derivatives
    (relu: the few pre-activations that change sign within the step) and f32's
    rounding of the loss."""
    d = data(50, 33, 47, F32, seed=5)
    gen = torch.Generator().manual_seed(7)
    dirs = {k: torch.randn(d[k].shape, generator=gen).cuda() for k in ("x", "w", "bias")}
    s = 1e-3

    def loss(sign):
        y = ops.linear(d["x"] + sign * s * dirs["x"], d["w"] + sign * s * dirs["w"], bias=d["bias"] + sign * s * dirs["bias"],
                       act=act)
        return float((y.double() * d["dy"].double()).sum())

    _, pre = ops.linear(d["x"], d["w"], bias=d["bias"], act=act, save_pre=True)
    g = ops.linear_backward(d["dy"], d["x"], d["w"], pre=pre if act != "none" else None, act=act)
    along = sum(float((a.double() * dirs[k].double()).sum()) for a, k in zip(g, ("x", "w", "bias")))
    size = sum(float((a.double() * dirs[k].double()).square().sum()) for a, k in zip(g, ("x", "w", "bias"))) ** 0.5
    assert abs((loss(1) - loss(-1)) / (2 * s) - along) <= 2e-3 * (abs(along) + 10 * size)


def test_graph_replays(ops):
    d = data(2000, 100, 60, BF16)
    args = (d["dy"], d["x"], d["w"])
    ops.linear_backward(*args, pre=d["pre"], act="silu")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.linear_backward(*args, pre=d["pre"], act="silu")
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = ops.linear_backward(*args, pre=d["pre"], act="silu")
        y = ops.linear(d["x"], d["w"], bias=d["bias"], act="gelu")
    for k in range(4):
        d["x"].mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, ops.linear_backward(*args, pre=d["pre"], act="silu")):
            assert torch.equal(a, b), k
        assert torch.equal(y, ops.linear(d["x"], d["w"], bias=d["bias"], act="gelu")), k
